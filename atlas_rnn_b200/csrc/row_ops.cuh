// Device helpers of the row operators (scan, convolution, sampling, distillation): packed fp32
// arithmetic, exponentials, whole-vector row accesses, transposed reductions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace atlas {
namespace ss {

constexpr float kLog2e = 1.4426950408889634f;

using f2 = unsigned long long;  // two fp32 in one 64-bit register (packed FMA)
__device__ __forceinline__ f2 pk(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 up(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ f2 ex2_2(f2 x) {
  const float2 v = up(x);
  return pk(ex2(v.x), ex2(v.y));
}

// log(1 + e^x) = max(x, 0) + log1p(e^-|x|), the logarithm by its series in s = e / (2 + e) <= 1/3:
// log1p(e) = 2 atanh(s) = 2 s (1 + s^2/3 + s^4/5 + ...); after s^12/13 the rest is below 2e-8 of it.
__device__ __forceinline__ float softplus(float x) {
  const float e = ex2(-fabsf(x) * kLog2e);
  const float s = e * rcp(2.f + e), q = s * s;
  float p = fmaf(q, 1.f / 13.f, 1.f / 11.f);
  p = fmaf(p, q, 1.f / 9.f);
  p = fmaf(p, q, 1.f / 7.f);
  p = fmaf(p, q, 1.f / 5.f);
  p = fmaf(p, q, 1.f / 3.f);
  p = fmaf(p, q, 1.f);
  const float r = fmaf(2.f * s, p, fmaxf(x, 0.f));
  return x != x ? x : r;
}
// 1 / (1 + e^-x); e^-x = inf gives 0.
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-x * kLog2e)); }

// W neighbouring elements of one row.
template <class IO, int W>
struct alignas(W * sizeof(IO)) Vec {
  IO v[W];
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float& o, float x) { o = x; }
__device__ __forceinline__ void from_f(__nv_bfloat16& o, float x) { o = __float2bfloat16_rn(x); }

// Elements c .. c + W - 1 of a row, 0 where c + i >= n.
template <class IO, int W>
__device__ __forceinline__ Vec<IO, W> load_row(const IO* p, int c, int n, int vec) {
  Vec<IO, W> r;
  if (vec && c + W <= n) return *reinterpret_cast<const Vec<IO, W>*>(p + c);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (c + i < n) r.v[i] = p[c + i];
    else from_f(r.v[i], 0.f);
  }
  return r;
}
template <class IO, int W>
__device__ __forceinline__ void store_row(IO* p, int c, int n, int vec, const Vec<IO, W>& r) {
  if (vec && c + W <= n) {
    *reinterpret_cast<Vec<IO, W>*>(p + c) = r;
    return;
  }
#pragma unroll
  for (int i = 0; i < W; ++i)
    if (c + i < n) p[c + i] = r.v[i];
}
template <class IO, int W>
__device__ __forceinline__ Vec<IO, W> zero_row() {
  Vec<IO, W> r;
#pragma unroll
  for (int i = 0; i < W; ++i) from_f(r.v[i], 0.f);
  return r;
}

// Sums over L lanes whose index differs in the bits L/2 .. 1 times `stride`: p[i] over all of them,
// lane k (its L-lane index) receives value k's sum in p[0]. L - 1 shuffles for L values.
template <int L, int STRIDE>
__device__ __forceinline__ void reduce_scatter(float* p, int lane) {
#pragma unroll
  for (int o = L / 2; o >= 1; o >>= 1) {
    const bool hi = lane & (o * STRIDE);
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = hi ? p[i + o] : p[i], send = hi ? p[i] : p[i + o];
      p[i] = keep + __shfl_xor_sync(0xffffffffu, send, o * STRIDE);
    }
  }
}

__device__ __forceinline__ int64_t row_len(const int* len, int b, int64_t T) {
  if (!len) return T;
  const int64_t l = len[b];
  return l < 0 ? 0 : (l > T ? T : l);
}

}  // namespace ss
}  // namespace atlas
