// Causal depthwise convolution with bias, SiLU and a carried state, forward and backward:
//   pre_t = bias + sum_j w[c,j] x[t + j - (K-1)],  y_t = silu(pre_t) or pre_t,
// steps before the sequence from the state [B, K-1, C]. Beside dwconv.cuh (three centred convolutions of one input) this
// is the one in front of the selective scan. A thread owns W neighbouring channels (8 bytes of bf16, 16 of fp32) and a
// run of steps, its taps and window in registers; a warp's lanes take neighbouring channel groups, so each load is a
// contiguous row segment, kConvU steps of them in flight. HBM-bound: the forward reads x once (plus K - 1 steps a run) and writes
// y; the backward reads x and dy, recomputes pre for the activation's slope and writes dx:
//   dp_t = dy_t act'(pre_t),  dx_s = sum_j w[j] dp_{s + K-1 - j},  dw[j] = sum_t dp_t x[t + j - (K-1)],  dbias = sum_t dp_t.
// Weight gradients: per-thread sums over the run, added over the CTA's four runs in shared memory, one record a CTA,
// records added in order by k_causal_conv_dw (no atomics: the same inputs give the same bits).
#pragma once
#include "row_ops.cuh"

namespace atlas {
namespace cc {

using ss::from_f;
using ss::load_row;
using ss::row_len;
using ss::sigmoid;
using ss::store_row;
using ss::to_f;
using ss::Vec;
using ss::zero_row;

constexpr int kConvWarps = 4;  // runs per CTA
constexpr int kConvU = 8;      // steps loaded ahead

struct ConvArgs {
  const void *x, *init, *dy, *d_final;
  int64_t x_sb, x_st, dy_sb, dy_st;
  const float *w, *bias;
  const int* len;
  void *y, *final_state, *dx, *d_init;
  float* part;  // [B * ygrid, C, K + 1]: dw, dbias of a CTA's steps
  int64_t T, C;
  int run, ygrid, silu, vec;  // steps per thread; CTAs along the time axis
};

// step t of the row (t >= -(K-1)), the state where t < 0
template <int K, class IO, int W>
__device__ __forceinline__ Vec<IO, W> step_row(const ConvArgs& a, const IO* x, const IO* init, int64_t t, int64_t c,
                                               int nc) {
  if (t >= 0) return load_row<IO, W>(x + t * a.x_st + c, 0, nc, a.vec);
  if (init) return load_row<IO, W>(init + (t + K - 1) * a.C + c, 0, nc, a.vec);
  return zero_row<IO, W>();
}

// grid (channel blocks, batch x time CTAs)
template <int K, class IO, int W>
__global__ void __launch_bounds__(32 * kConvWarps) k_causal_conv_fwd(const ConvArgs a) {
  const int64_t c = ((int64_t)blockIdx.y * 32 + (threadIdx.x & 31)) * W;
  if (c >= a.C) return;
  const int nc = a.C - c < W ? (int)(a.C - c) : W;
  const int64_t b = blockIdx.x / a.ygrid, r = (blockIdx.x - b * a.ygrid) * kConvWarps + (threadIdx.x >> 5);
  const int64_t len = row_len(a.len, (int)b, a.T);
  const int64_t t0 = r * a.run, t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
  const IO* x = (const IO*)a.x + b * a.x_sb;
  const IO* init = a.init ? (const IO*)a.init + b * (K - 1) * a.C : nullptr;
  if (r == 0) {  // the last K - 1 inputs of the row
    IO* f = (IO*)a.final_state + b * (K - 1) * a.C + c;
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
      store_row<IO, W>(f + i * a.C, 0, nc, a.vec, step_row<K, IO, W>(a, x, init, len + i - (K - 1), c, nc));
  }
  if (t0 >= a.T) return;
  IO* y = (IO*)a.y + b * a.T * a.C + c;
  float w[K][W], bias[W], win[K][W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    bias[i] = a.bias && i < nc ? a.bias[c + i] : 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = i < nc ? a.w[(c + i) * K + j] : 0.f;
  }
  if (t0 < len) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      const Vec<IO, W> v = step_row<K, IO, W>(a, x, init, t0 + j - (K - 1), c, nc);
#pragma unroll
      for (int i = 0; i < W; ++i) win[j][i] = to_f(v.v[i]);
    }
  }
  for (int64_t t = t0; t < t1; t += kConvU) {
    Vec<IO, W> in[kConvU];
#pragma unroll
    for (int k = 0; k < kConvU; ++k)
      in[k] = t + k < t1 && t + k < len ? load_row<IO, W>(x + (t + k) * a.x_st + c, 0, nc, a.vec) : zero_row<IO, W>();
#pragma unroll
    for (int k = 0; k < kConvU; ++k) {
      if (t + k >= t1) break;
      Vec<IO, W> o = zero_row<IO, W>();
      if (t + k < len) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          win[K - 1][i] = to_f(in[k].v[i]);
          float s = bias[i];
#pragma unroll
          for (int j = 0; j < K; ++j) s = fmaf(w[j][i], win[j][i], s);
          if (a.silu) s *= sigmoid(s);
          from_f(o.v[i], s);
#pragma unroll
          for (int j = 0; j < K - 1; ++j) win[j][i] = win[j + 1][i];
        }
      }
      store_row<IO, W>(y + (t + k) * a.C, 0, nc, a.vec, o);
    }
  }
}

template <int K, class IO, int W>
__global__ void __launch_bounds__(32 * kConvWarps) k_causal_conv_bwd(const ConvArgs a) {
  __shared__ float s_red[kConvWarps][32][W * (K + 1) + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.y * 32 + lane) * W;
  const int nc = c >= a.C ? 0 : a.C - c < W ? (int)(a.C - c) : W;
  const int64_t b = blockIdx.x / a.ygrid, yb = blockIdx.x - b * a.ygrid, r = yb * kConvWarps + warp;
  const int64_t len = row_len(a.len, (int)b, a.T);
  const int64_t t0 = r * a.run, t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
  float acc[K][W], accb[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    accb[i] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) acc[j][i] = 0.f;
  }
  if (nc > 0 && t0 < a.T) {
    const IO* x = (const IO*)a.x + b * a.x_sb;
    const IO* dy = (const IO*)a.dy + b * a.dy_sb + c;
    const IO* init = a.init ? (const IO*)a.init + b * (K - 1) * a.C : nullptr;
    const IO* df = a.d_final ? (const IO*)a.d_final + b * (K - 1) * a.C + c : nullptr;
    IO* dx = (IO*)a.dx + b * a.T * a.C + c;
    IO* di = a.d_init ? (IO*)a.d_init + b * (K - 1) * a.C + c : nullptr;
    float w[K][W], bias[W], win[K][W], dp[K][W];  // dp[j]: step t - j
#pragma unroll
    for (int i = 0; i < W; ++i) {
      bias[i] = a.bias && i < nc ? a.bias[c + i] : 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        w[j][i] = i < nc ? a.w[(c + i) * K + j] : 0.f;
        dp[j][i] = 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      const Vec<IO, W> v = t0 + j - (K - 1) < len ? step_row<K, IO, W>(a, x, init, t0 + j - (K - 1), c, nc)
                                                  : zero_row<IO, W>();
#pragma unroll
      for (int i = 0; i < W; ++i) win[j][i] = to_f(v.v[i]);
    }
    const int64_t tend = t1 + K - 1;
    for (int64_t t = t0; t < tend; t += kConvU) {
      Vec<IO, W> in[kConvU], up[kConvU];
#pragma unroll
      for (int k = 0; k < kConvU; ++k) {
        const bool live = t + k < tend && t + k < len;
        in[k] = live ? load_row<IO, W>(x + (t + k) * a.x_st + c, 0, nc, a.vec) : zero_row<IO, W>();
        up[k] = live ? load_row<IO, W>(dy + (t + k) * a.dy_st, 0, nc, a.vec) : zero_row<IO, W>();
      }
#pragma unroll
      for (int k = 0; k < kConvU; ++k) {
        if (t + k >= tend) break;
        const int64_t s = t + k - (K - 1);
        Vec<IO, W> extra = zero_row<IO, W>();  // the gradient of the final state, where step s is in it
        const int64_t at = s - (len - (K - 1));
        if (df && at >= 0 && at < K - 1) extra = load_row<IO, W>(df + at * a.C, 0, nc, a.vec);
        Vec<IO, W> o;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          win[K - 1][i] = to_f(in[k].v[i]);
          float d = to_f(up[k].v[i]);
          if (a.silu) {
            float p = bias[i];
#pragma unroll
            for (int j = 0; j < K; ++j) p = fmaf(w[j][i], win[j][i], p);
            const float sg = sigmoid(p);
            // slope of silu; where e^-p overflows sg is 0 and so is the slope
            d *= sg * fmaf(p, 1.f - sg, 1.f);
          }
          if (t + k >= len) d = 0.f;
#pragma unroll
          for (int j = K - 1; j > 0; --j) dp[j][i] = dp[j - 1][i];
          dp[0][i] = d;
          if (t + k < t1) {
            accb[i] += d;
#pragma unroll
            for (int j = 0; j < K; ++j) acc[j][i] = fmaf(d, win[j][i], acc[j][i]);
          }
          float g = to_f(extra.v[i]);
#pragma unroll
          for (int j = 0; j < K; ++j) g = fmaf(w[j][i], dp[j][i], g);
          from_f(o.v[i], s < len ? g : 0.f);
#pragma unroll
          for (int j = 0; j < K - 1; ++j) win[j][i] = win[j + 1][i];
        }
        if (s >= t0 && s < t1) store_row<IO, W>(dx + s * a.C, 0, nc, a.vec, o);
        else if (s < 0 && di) store_row<IO, W>(di + (s + K - 1) * a.C, 0, nc, a.vec, o);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) s_red[warp][lane][i * (K + 1) + j] = acc[j][i];
    s_red[warp][lane][i * (K + 1) + K] = accb[i];
  }
  __syncthreads();
  // record of this CTA: 32 W channels x (K + 1), channel-major like w
  const int64_t cb = (int64_t)blockIdx.y * 32 * W, left = a.C - cb;
  const int n = (int)(left < 32 * W ? left : 32 * W) * (K + 1);
  float* out = a.part + ((int64_t)blockIdx.x * a.C + cb) * (K + 1);
  for (int e = threadIdx.x; e < n; e += 32 * kConvWarps) {
    const int ln = e / (W * (K + 1)), k = e - ln * (W * (K + 1));
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < kConvWarps; ++q) s += s_red[q][ln][k];
    out[e] = s;
  }
}

// dw [C, K] and dbias [C]: records added in order, 8 slices of them a value.
__global__ void __launch_bounds__(256) k_causal_conv_dw(const float* part, float* dw, float* dbias, int64_t n,
                                                        int K, int64_t records) {
  __shared__ float s_red[8][32];
  const int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int sl = threadIdx.x >> 5;
  float s = 0.f;
  if (i < n) {
    const int64_t lo = records * sl / 8, hi = records * (sl + 1) / 8;
#pragma unroll 8
    for (int64_t r = lo; r < hi; ++r) s += part[r * n + i];
  }
  s_red[sl][threadIdx.x & 31] = s;
  __syncthreads();
  if (sl == 0 && i < n) {
#pragma unroll
    for (int q = 1; q < 8; ++q) s += s_red[q][threadIdx.x];
    const int64_t c = i / (K + 1);
    const int j = (int)(i - c * (K + 1));
    if (j < K) dw[c * K + j] = s;
    else if (dbias) dbias[c] = s;
  }
}

}  // namespace cc
}  // namespace atlas
