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
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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
  float p = fmaf(q, 2.f / 13.f, 2.f / 11.f);
  p = fmaf(p, q, 2.f / 9.f);
  p = fmaf(p, q, 2.f / 7.f);
  p = fmaf(p, q, 2.f / 5.f);
  p = fmaf(p, q, 2.f / 3.f);
  p = fmaf(p, q, 2.f);
  return fmaf(s, p, fmaxf(x, 0.f));  // a NaN comes through s
}
// 1 / (1 + e^-x); e^-x = inf gives 0.
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-x * kLog2e)); }

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float& o, float x) { o = x; }
__device__ __forceinline__ void from_f(__nv_bfloat16& o, float x) { o = __float2bfloat16_rn(x); }

__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 both(float x) { return pk(x, x); }
__device__ __forceinline__ f2 rcp_2(f2 x) {
  const float2 v = up(x);
  return pk(rcp(v.x), rcp(v.y));
}
__device__ __forceinline__ f2 sigmoid_2(f2 x) { return rcp_2(add2(both(1.f), ex2_2(mul2(x, both(-kLog2e))))); }
// softplus() of both halves: plain FMAs, whose constants are immediates (packed ones would take them from registers)
__device__ __forceinline__ f2 softplus_2(f2 x) {
  const float2 v = up(x);
  return pk(softplus(v.x), softplus(v.y));
}

// Two neighbouring elements as fp32, and back.
__device__ __forceinline__ f2 ld2(const float* p) { return *reinterpret_cast<const f2*>(p); }
__device__ __forceinline__ f2 ld2(const __nv_bfloat16* p) {
  const unsigned v = *reinterpret_cast<const unsigned*>(p);  // a bf16 is the high half of its fp32
  return pk(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ void st2(float* p, f2 v) { *reinterpret_cast<f2*>(p) = v; }
__device__ __forceinline__ void st2(__nv_bfloat16* p, f2 v) {
  const float2 x = up(v);
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x.x, x.y);
}

// SIZE (8 or 16) bytes to shared memory in the background: the first `bytes` from src, zeros behind them.
template <int SIZE>
__device__ __forceinline__ void cp_piece(void* dst, const void* src, int bytes) {
  const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
  if constexpr (SIZE == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// A warp's feed of [ROWS, W] tiles out of rows `stride` elements apart into shared memory, zeros past n columns and past
// the rows left. `vec`: rows are 16-byte aligned and go by cp.async, each lane its own column piece (16 bytes, or the
// row's 8) of every 32 / PER-th row (commit and wait are the caller's); otherwise element by element.
template <class IO, int ROWS, int W>
struct Feed {
  static constexpr int E = W * (int)sizeof(IO) < 16 ? W : 16 / (int)sizeof(IO), PER = W / E, STEP = 32 / PER;
  static_assert(W % E == 0 && E * sizeof(IO) >= 8 && PER <= 32 && 32 % PER == 0, "whole pieces");
  const IO* p;  // vec: the lane's piece of the tile's first row of its own; else the tile's first row
  int bytes;    // vec: of the lane's pieces; else the columns
  __device__ __forceinline__ Feed(const IO* src, int64_t stride, int n, int vec, int lane) {
    if (vec) {
      const int k = n - lane % PER * E;
      p = src + lane / PER * stride + lane % PER * E;
      bytes = (k < 0 ? 0 : k > E ? E : k) * (int)sizeof(IO);
      if (bytes == 0) p = src;
    } else {
      p = src;
      bytes = n;
    }
  }
  __device__ __forceinline__ void vectors(IO* dst, int64_t stride, int rows, int lane) const {
#pragma unroll
    for (int i = 0; i < ROWS; i += STEP) {
      const int r = lane / PER + i;
      if (ROWS % STEP != 0 && r >= ROWS) break;
      cp_piece<E * (int)sizeof(IO)>(dst + r * W + lane % PER * E, p + i * stride, r < rows ? bytes : 0);
    }
  }
  __device__ __forceinline__ void elements(IO* dst, int64_t stride, int rows, int lane) const {
#pragma unroll 4
    for (int at = lane; at < ROWS * W; at += 32) {
      const int r = at / W, c = at % W;
      if (r < rows && c < bytes) dst[at] = p[r * stride + c];
      else from_f(dst[at], 0.f);
    }
  }
};

// W neighbouring elements of one row.
template <class IO, int W>
struct alignas(W * sizeof(IO)) Vec {
  IO v[W];
};
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

// Sums of V values over L lanes (index bits of weight STRIDE, 2 STRIDE, ..): the lane of L-lane index k keeps values
// k V/L .. in p[0 .. V/L - 1]. V - V/L exchanges instead of V log2(L).
template <int V, int L, int STRIDE>
__device__ __forceinline__ void reduce_part(float* p, int lane) {
  static_assert(V >= L, "a value for every lane");
  int n = V;
#pragma unroll
  for (int o = L / 2; o >= 1; o >>= 1) {
    n >>= 1;
    const bool hi = lane & (o * STRIDE);
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      if (i < n) {
        const float keep = hi ? p[i + n] : p[i], send = hi ? p[i] : p[i + n];
        p[i] = keep + __shfl_xor_sync(0xffffffffu, send, o * STRIDE);
      }
  }
}
// The same over V pairs, added two at a time; the last halving splits a pair where L = 2 V (then p[0]'s low half).
template <int V, int L, int STRIDE>
__device__ __forceinline__ void reduce_pairs(f2* p, int lane) {
  static_assert(2 * V >= L, "a value for every lane");
  int n = V;
#pragma unroll
  for (int o = L / 2; o >= 1; o >>= 1) {
    const bool hi = lane & (o * STRIDE);
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < (V + 1) / 2; ++i)
        if (i < n) {
          const f2 keep = hi ? p[i + n] : p[i], send = hi ? p[i] : p[i + n];
          p[i] = add2(keep, __shfl_xor_sync(0xffffffffu, send, o * STRIDE));
        }
    } else {
      const float2 v = up(p[0]);
      const float keep = hi ? v.y : v.x, send = hi ? v.x : v.y;
      p[0] = both(keep + __shfl_xor_sync(0xffffffffu, send, o * STRIDE));
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
