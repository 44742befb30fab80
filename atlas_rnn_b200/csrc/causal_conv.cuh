// Causal depthwise convolution with bias, SiLU and a carried state, forward and backward:
//   pre_t = bias + sum_j w[c,j] x[t + j - (K-1)],  y_t = silu(pre_t) or pre_t,
// steps before the sequence from the state [B, K-1, C]. Beside dwconv.cuh (three centred convolutions of one input) this
// is the one in front of the selective scan. A thread owns W neighbouring channels (8 bytes of bf16, 16 of fp32) and a
// run of steps, its taps and window in registers; a warp's lanes take neighbouring channel groups, so each load is a
// contiguous row segment, kConvU steps of them in flight. HBM-bound: the forward reads x once (plus K - 1 steps a run) and writes
// y; the backward reads x and dy, recomputes pre for the activation's slope and writes dx:
// B 4, T 8192, C 1536, K 4, bf16: forward 51 us (3.9 TB/s), backward 100 (3.0 TB/s), both waiting for loads with the warps
// that their registers leave. Results are rounded to the rows' type once, when they are written.
//   dp_t = dy_t act'(pre_t),  dx_s = sum_j w[j] dp_{s + K-1 - j},  dw[j] = sum_t dp_t x[t + j - (K-1)],  dbias = sum_t dp_t.
// Weight gradients: per-thread sums over the run, added over the CTA's four runs in shared memory, one record a CTA,
// records added in order by k_causal_conv_dw (no atomics: the same inputs give the same bits).
#pragma once
#include "row_ops.cuh"

namespace atlas {
namespace cc {

using ss::add2;
using ss::both;
using ss::ex2_2;
using ss::f2;
using ss::fma2;
using ss::from_f;
using ss::ld2;
using ss::mul2;
using ss::pk;
using ss::row_len;
using ss::sigmoid_2;
using ss::st2;
using ss::to_f;
using ss::up;
using ss::Vec;

constexpr int kConvWarps = 4;  // runs per CTA
constexpr int kConvU = 8;      // steps in flight
constexpr int kConvG = 4;      // backward of 16-bit rows: steps of a group

struct ConvArgs {
  const void *x, *init, *dy, *d_final;
  int64_t x_sb, x_st, dy_sb, dy_st;
  const float *w, *bias;
  const int* len;
  void *y, *final_state, *dx, *d_init;
  float* part;  // [B * ygrid, C, K + 1]: dw, dbias of a CTA's steps
  int64_t T, C, rows;
  int run, ygrid, silu, vec;  // steps per thread; CTAs along the time axis
};

// W channels of a row as pairs: whole vectors where `fast`, else those below nc one by one.
template <class IO, int W>
struct Row {
  f2 v[W / 2];
};
template <class IO, int W>
__device__ __forceinline__ Row<IO, W> widen(const Vec<IO, W>& r) {
  Row<IO, W> o;
#pragma unroll
  for (int i = 0; i < W / 2; ++i) o.v[i] = ld2(&r.v[2 * i]);
  return o;
}
template <class IO, int W>
__device__ __forceinline__ Row<IO, W> load(const IO* p, int nc, bool fast) {
  if (fast) return widen<IO, W>(*reinterpret_cast<const Vec<IO, W>*>(p));
  Row<IO, W> o;
#pragma unroll
  for (int i = 0; i < W / 2; ++i) o.v[i] = pk(2 * i < nc ? to_f(p[2 * i]) : 0.f, 2 * i + 1 < nc ? to_f(p[2 * i + 1]) : 0.f);
  return o;
}
template <class IO, int W>
__device__ __forceinline__ void store(IO* p, const Row<IO, W>& r, int nc, bool fast) {
  if (fast) {
    Vec<IO, W> o;
#pragma unroll
    for (int i = 0; i < W / 2; ++i) st2(&o.v[2 * i], r.v[i]);
    *reinterpret_cast<Vec<IO, W>*>(p) = o;
    return;
  }
#pragma unroll
  for (int i = 0; i < W; ++i)
    if (i < nc) from_f(p[i], i % 2 ? up(r.v[i / 2]).y : up(r.v[i / 2]).x);
}
template <class IO, int W>
__device__ __forceinline__ Row<IO, W> zeros() {
  Row<IO, W> o;
#pragma unroll
  for (int i = 0; i < W / 2; ++i) o.v[i] = 0;
  return o;
}

// A thread's place: W channels from c, steps t0 .. t0 + n - 1 of row b, of which `live` are before the row's length
// (more or fewer than n, or none: the values beside the run matter only up to K away).
template <int K, class IO, int W>
struct Run {
  int64_t b, c, t0, len;
  int r, n, live, nc;
  bool fast;
  const IO *x, *init;
  __device__ __forceinline__ explicit Run(const ConvArgs& a) {
    c = ((int64_t)blockIdx.y * 32 + (threadIdx.x & 31)) * W;
    nc = c >= a.C ? 0 : a.C - c < W ? (int)(a.C - c) : W;
    b = blockIdx.x / a.ygrid;
    r = (int)(blockIdx.x - b * a.ygrid) * kConvWarps + (threadIdx.x >> 5);
    len = row_len(a.len, (int)b, a.T);
    t0 = (int64_t)r * a.run;
    n = a.T - t0 < a.run ? (a.T - t0 < 0 ? 0 : (int)(a.T - t0)) : a.run;
    const int64_t l = len - t0;
    live = l < -K ? -K : l > a.run + K ? a.run + K : (int)l;
    fast = a.vec && nc == W;
    x = (const IO*)a.x + b * a.x_sb + c;
    init = a.init ? (const IO*)a.init + b * (K - 1) * a.C + c : nullptr;
  }
  // step t of the row (t >= -(K - 1)), the state where t < 0
  __device__ __forceinline__ Row<IO, W> at(const ConvArgs& a, int64_t t) const {
    if (t >= 0) return load<IO, W>(x + t * a.x_st, nc, fast);
    if (init) return load<IO, W>(init + (t + K - 1) * a.C, nc, fast);
    return zeros<IO, W>();
  }
  __device__ __forceinline__ void taps(const ConvArgs& a, f2 (&w)[K][W / 2], f2 (&bias)[W / 2]) const {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const bool o0 = 2 * i < nc, o1 = 2 * i + 1 < nc;
      const int64_t k = c + 2 * i;
      bias[i] = pk(a.bias && o0 ? a.bias[k] : 0.f, a.bias && o1 ? a.bias[k + 1] : 0.f);
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][i] = pk(o0 ? a.w[k * K + j] : 0.f, o1 ? a.w[(k + 1) * K + j] : 0.f);
    }
  }
};

// grid (batch x time CTAs, channel blocks)
template <int K, class IO, int W>
__global__ void __launch_bounds__(32 * kConvWarps) k_causal_conv_fwd(const ConvArgs a) {
  constexpr int P = W / 2;
  const Run<K, IO, W> q(a);
  if (q.nc == 0) return;
  if (q.r == 0) {  // the last K - 1 inputs of the row
    IO* f = (IO*)a.final_state + q.b * (K - 1) * a.C + q.c;
#pragma unroll
    for (int i = 0; i < K - 1; ++i) store<IO, W>(f + i * a.C, q.at(a, q.len + i - (K - 1)), q.nc, q.fast);
  }
  if (q.n == 0) return;
  IO* y = (IO*)a.y + (q.b * a.T + q.t0) * a.C + q.c;
  f2 w[K][P], bias[P], win[K][P];  // win[j]: step t + j - (K - 1)
  q.taps(a, w, bias);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const Row<IO, W> v = q.live > 0 ? q.at(a, q.t0 + j - (K - 1)) : zeros<IO, W>();
#pragma unroll
    for (int i = 0; i < P; ++i) win[j][i] = v.v[i];
  }
  auto step = [&](const Row<IO, W>& in) {
    Row<IO, W> o;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      win[K - 1][i] = in.v[i];
      f2 s = bias[i];
#pragma unroll
      for (int j = 0; j < K; ++j) s = fma2(w[j][i], win[j][i], s);
      o.v[i] = a.silu ? mul2(s, sigmoid_2(s)) : s;
#pragma unroll
      for (int j = 0; j < K - 1; ++j) win[j][i] = win[j + 1][i];
    }
    return o;
  };
  const IO* x = q.x + q.t0 * a.x_st;
  const int nl = q.n < q.live ? q.n : q.live;
  int t = 0;
  if (q.fast)
    for (; t + kConvU <= nl; t += kConvU) {
      Vec<IO, W> in[kConvU];
#pragma unroll
      for (int k = 0; k < kConvU; ++k) in[k] = *reinterpret_cast<const Vec<IO, W>*>(x + (t + k) * a.x_st);
#pragma unroll
      for (int k = 0; k < kConvU; ++k) store<IO, W>(y + (t + k) * a.C, step(widen<IO, W>(in[k])), W, true);
    }
#pragma unroll 2
  for (; t < nl; ++t) store<IO, W>(y + t * a.C, step(load<IO, W>(x + t * a.x_st, q.nc, q.fast)), q.nc, q.fast);
  for (; t < q.n; ++t) store<IO, W>(y + t * a.C, zeros<IO, W>(), q.nc, q.fast);
}

// One step (T = 1): a thread reads its channels' taps, and of R batch rows the K - 1 carried inputs and the new one, all in
// flight together, and writes y and the shifted states. FAST: whole vectors. grid (channel blocks, row blocks).
constexpr int kConvStepThr = 128;
template <int K, class IO, int W, int R, bool FAST>
__global__ void __launch_bounds__(kConvStepThr) k_causal_conv_step(const ConvArgs a) {
  constexpr int P = W / 2;
  const int64_t b0 = (int64_t)blockIdx.y * R, c = ((int64_t)blockIdx.x * kConvStepThr + threadIdx.x) * W;
  if (c >= a.C) return;
  const int nc = a.C - c < W ? (int)(a.C - c) : W;
  const int left = a.rows - b0 < R ? (int)(a.rows - b0) : R;
  auto raw = [&](const IO* p) {
    if (FAST) return *reinterpret_cast<const Vec<IO, W>*>(p);
    return ss::load_row<IO, W>(p, 0, nc, 0);
  };
  auto put = [&](IO* p, const Vec<IO, W>& r) {
    if (FAST) *reinterpret_cast<Vec<IO, W>*>(p) = r;
    else ss::store_row<IO, W>(p, 0, nc, 0, r);
  };
  const int64_t state = (K - 1) * a.C;
  const IO* init = a.init ? (const IO*)a.init + b0 * state + c : nullptr;
  const IO* x = (const IO*)a.x + b0 * a.x_sb + c;
  Vec<IO, W> v[R][K];
  int len[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t k = r < left ? r : 0;  // rows that exist
#pragma unroll
    for (int j = 0; j < K - 1; ++j) v[r][j] = init ? raw(init + k * state + j * a.C) : ss::zero_row<IO, W>();
    v[r][K - 1] = raw(x + k * a.x_sb);
    len[r] = a.len ? a.len[b0 + k] : 1;
  }
  float w[W][K], bias[W];
  if (FAST && W * K % 4 == 0) {  // the channels' taps lie side by side (alignment: `vec` asks for 16 bytes of w)
#pragma unroll
    for (int i = 0; i < W * K / 4 * 4; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(a.w + c * K + i);
      w[i / K][i % K] = t.x, w[(i + 1) / K][(i + 1) % K] = t.y, w[(i + 2) / K][(i + 2) % K] = t.z, w[(i + 3) / K][(i + 3) % K] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < K; ++j) w[i][j] = a.w[(FAST || i < nc ? c + i : c) * K + j];
  }
#pragma unroll
  for (int i = 0; i < W; ++i) bias[i] = a.bias ? a.bias[FAST || i < nc ? c + i : c] : 0.f;
  IO* f = (IO*)a.final_state + b0 * state + c;
  IO* y = (IO*)a.y + b0 * a.C + c;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= left) break;
    const bool live = len[r] > 0;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) put(f + r * state + j * a.C, live ? v[r][j + 1] : v[r][j]);
    Vec<IO, W> o;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      f2 s = pk(bias[2 * i], bias[2 * i + 1]);
#pragma unroll
      for (int j = 0; j < K; ++j) s = fma2(pk(w[2 * i][j], w[2 * i + 1][j]), ld2(&v[r][j].v[2 * i]), s);
      if (a.silu) s = mul2(s, sigmoid_2(s));
      st2(&o.v[2 * i], live ? s : 0);
    }
    put(y + r * a.C, o);
  }
}

template <int K, class IO, int W>
__global__ void __launch_bounds__(32 * kConvWarps) k_causal_conv_bwd(const ConvArgs a) {
  constexpr int P = W / 2;
  __shared__ float s_red[kConvWarps][32][W * (K + 1) + 1];
  const Run<K, IO, W> q(a);
  f2 acc[K][P], accb[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    accb[i] = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) acc[j][i] = 0;
  }
  if (q.nc > 0 && q.n > 0) {
    const IO* x = q.x + q.t0 * a.x_st;
    const IO* dy = (const IO*)a.dy + q.b * a.dy_sb + q.t0 * a.dy_st + q.c;
    const IO* df = a.d_final ? (const IO*)a.d_final + q.b * (K - 1) * a.C + q.c : nullptr;
    IO* dx = (IO*)a.dx + (q.b * a.T + q.t0) * a.C + q.c;
    IO* di = a.d_init && q.r == 0 ? (IO*)a.d_init + q.b * (K - 1) * a.C + q.c : nullptr;
    f2 w[K][P], bias[P], win[K][P], dp[K][P];  // dp[j]: the gradient of pre at step t - j
    q.taps(a, w, bias);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      const Row<IO, W> v = j - (K - 1) < q.live ? q.at(a, q.t0 + j - (K - 1)) : zeros<IO, W>();
#pragma unroll
      for (int i = 0; i < P; ++i) win[j][i] = v.v[i];
    }
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) dp[j][i] = 0;
    // one step; the gradient it completes is step t - (K - 1)'s. own: counts for dw
    auto step = [&](const Row<IO, W>& in, const Row<IO, W>& up_, bool own) {
      Row<IO, W> o;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        win[K - 1][i] = in.v[i];
        f2 d = up_.v[i];
        if (a.silu) {
          f2 p = bias[i];
#pragma unroll
          for (int j = 0; j < K; ++j) p = fma2(w[j][i], win[j][i], p);
          // slope of silu: sg (1 + p (1 - sg))
          const f2 sg = sigmoid_2(p);
          d = mul2(mul2(d, sg), fma2(p, fma2(sg, both(-1.f), both(1.f)), both(1.f)));
        }
#pragma unroll
        for (int j = K - 1; j > 0; --j) dp[j][i] = dp[j - 1][i];
        dp[0][i] = d;
        if (own) {
          accb[i] = add2(accb[i], d);
#pragma unroll
          for (int j = 0; j < K; ++j) acc[j][i] = fma2(d, win[j][i], acc[j][i]);
        }
        f2 g = mul2(w[0][i], dp[0][i]);
#pragma unroll
        for (int j = 1; j < K; ++j) g = fma2(w[j][i], dp[j][i], g);
        o.v[i] = g;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) win[j][i] = win[j + 1][i];
      }
      return o;
    };
    // a step anywhere: past the length, before the run, the gradient of the final state
    auto edge = [&](int t) {
      const bool on = t < q.live;
      Row<IO, W> o = step(on ? load<IO, W>(x + t * a.x_st, q.nc, q.fast) : zeros<IO, W>(),
                          on ? load<IO, W>(dy + t * a.dy_st, q.nc, q.fast) : zeros<IO, W>(), on && t < q.n);
      const int s = t - (K - 1), at = s - (q.live - (K - 1));
      if (s >= q.live) o = zeros<IO, W>();
      else if (df && at >= 0) {
        const Row<IO, W> e = load<IO, W>(df + at * a.C, q.nc, q.fast);
#pragma unroll
        for (int i = 0; i < P; ++i) o.v[i] = add2(o.v[i], e.v[i]);
      }
      if (s >= 0 && s < q.n) store<IO, W>(dx + s * a.C, o, q.nc, q.fast);
      else if (s < 0 && di) store<IO, W>(di + (s + K - 1) * a.C, o, q.nc, q.fast);
    };
    const int nl = q.n < q.live ? q.n : q.live;
    int t = 0;
#pragma unroll 1
    for (; t < K - 1; ++t) edge(t);  // complete gradients of the run before, or of the initial state
    if (sizeof(IO) == 2 && q.fast) {
      // groups of kConvG steps, the next one on its way meanwhile (B 4, T 8192, C 1536: 101 us, without 117; fp32 rows, which
      // take twice the registers: 158 and 116)
      Vec<IO, W> in[kConvG], up_[kConvG], in2[kConvG], up2[kConvG];
      auto fetch = [&](int at, Vec<IO, W>(&i)[kConvG], Vec<IO, W>(&u)[kConvG]) {
#pragma unroll
        for (int k = 0; k < kConvG; ++k) {
          i[k] = *reinterpret_cast<const Vec<IO, W>*>(x + (at + k) * a.x_st);
          u[k] = *reinterpret_cast<const Vec<IO, W>*>(dy + (at + k) * a.dy_st);
        }
      };
      auto walk = [&](int at, const Vec<IO, W>(&i)[kConvG], const Vec<IO, W>(&u)[kConvG]) {
#pragma unroll
        for (int k = 0; k < kConvG; ++k)
          store<IO, W>(dx + (at + k - (K - 1)) * a.C, step(widen<IO, W>(i[k]), widen<IO, W>(u[k]), true), W, true);
      };
      if (t + kConvG <= nl) fetch(t, in, up_);
      for (; t + 2 * kConvG <= nl; t += 2 * kConvG) {
        fetch(t + kConvG, in2, up2);
        walk(t, in, up_);
        if (t + 3 * kConvG <= nl) fetch(t + 2 * kConvG, in, up_);
        walk(t + kConvG, in2, up2);
      }
      if (t + kConvG <= nl) {
        walk(t, in, up_);
        t += kConvG;
      }
    } else if (q.fast) {
      for (; t + kConvU <= nl; t += kConvU) {
        Vec<IO, W> in[kConvU], up_[kConvU];
#pragma unroll
        for (int k = 0; k < kConvU; ++k) {
          in[k] = *reinterpret_cast<const Vec<IO, W>*>(x + (t + k) * a.x_st);
          up_[k] = *reinterpret_cast<const Vec<IO, W>*>(dy + (t + k) * a.dy_st);
        }
#pragma unroll
        for (int k = 0; k < kConvU; ++k)
          store<IO, W>(dx + (t + k - (K - 1)) * a.C, step(widen<IO, W>(in[k]), widen<IO, W>(up_[k]), true), W, true);
      }
    }
#pragma unroll 1
    for (; t < q.n + K - 1; ++t) edge(t);
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
    auto half = [&](f2 v) { return i % 2 ? up(v).y : up(v).x; };
#pragma unroll
    for (int j = 0; j < K; ++j) s_red[threadIdx.x >> 5][threadIdx.x & 31][i * (K + 1) + j] = half(acc[j][i / 2]);
    s_red[threadIdx.x >> 5][threadIdx.x & 31][i * (K + 1) + K] = half(accb[i / 2]);
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
    for (int u = 0; u < kConvWarps; ++u) s += s_red[u][ln][k];
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
