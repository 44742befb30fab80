// Distillation from a teacher's top logits, forward and backward. Per row, with the teacher's entries (value v_k, token i_k;
// entries with i_k outside 0 .. V-1, or -inf or NaN values, are absent) and the student's logits x:
//   p = softmax(v / tau) over the entries,  q = softmax(x / tau) over the vocabulary,
//   loss = tau^2 sum_k p_k (log p_k - log q_{i_k}),   d loss / d x_j = tau (q_j - sum_{k: i_k = j} p_k)
// (tokens may repeat), and 0 for a row without entries. The forward reads the logits once with a running maximum m and
// sum s = sum 2^(c (x - m)), c = log2(e) / tau, so log2 q_j = c (x_j - m) - log2 s; the difference is taken first, so that
// logits of any size keep their distances. The backward reads them again, writes tau g q everywhere, and then the
// entries' own values.
// HBM-bound: 3 x rows x V elements over both (8192 x 32000, bf16: forward 103 us, 5.1 TB/s, with the special-function unit
// 70% busy; backward 172 us, 6.1 TB/s). Few rows are split over a cluster of CTAs.
#pragma once
#include <cooperative_groups.h>

#include "row_ops.cuh"

namespace atlas {
namespace dst {

namespace cg = cooperative_groups;
constexpr int kMaxK = 1024;
constexpr int kMarks = 512;  // words of a bitmap of tokens, by their low bits
// Short rows of few entries: a warp a row, 4 rows a CTA, since the start of a CTA costs more than such a row (32768 x 256,
// bf16, 20 entries: forward 25 us, backward 29; a CTA a row 50 and 67).
constexpr int kShortV = 1024, kShortK = 128, kShortRows = 4;

struct DistillArgs {
  const void* logits;
  int64_t stride;
  const float* values;     // [rows, K]
  const int64_t* indices;  // [rows, K]
  float* loss;             // [rows]
  float* valid;            // [rows] 1 with entries, 0 without
  float* stats;            // [rows, 4]: m and log2 s of the student; maximum and sum of the teacher (0: no entries)
  const float* dloss;
  void* dlogits;  // [rows, V]
  int V, K, split;
  int rows;
  float tau;
};

template <class T, class F>
__device__ __forceinline__ T warp_reduce(T v, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float fmax_op(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float add_op(float a, float b) { return a + b; }

// Elements before the first 16-byte boundary of a row (all n of them if it lies behind).
template <class IO>
__device__ __forceinline__ int head_of(const IO* p, int n) {
  const int h = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(IO);
  return h < n ? h : n;
}
// Largest of a vector's elements (NaN is none).
__device__ __forceinline__ float vec_max(const ss::Vec<float, 4>& r) {
  return fmaxf(fmaxf(r.v[0], r.v[1]), fmaxf(r.v[2], r.v[3]));
}
__device__ __forceinline__ float vec_max(const ss::Vec<__nv_bfloat16, 8>& r) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(r.v);
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Value and token of entry k, -inf where it is absent.
__device__ __forceinline__ float entry(const DistillArgs& a, int64_t row, int k, int64_t& token) {
  token = a.indices[row * a.K + k];
  const float v = a.values[row * a.K + k];
  return token >= 0 && token < a.V && v > -INFINITY ? v : -INFINITY;
}
// exp((v - top) / tau) of a present entry, by the row's maximum; 0 of an absent one (-inf, also where top is)
__device__ __forceinline__ float weight(float v, float top, float c) {
  if (!(v > -INFINITY)) return 0.f;
  return v == top ? 1.f : exp2f((v - top) * c);
}

// grid rows x cluster; NT threads a row, RPC rows a CTA (then one warp a row)
template <class IO, int NT, int RPC>
__global__ void __launch_bounds__(NT * RPC) k_distill_fwd(const DistillArgs a) {
  constexpr int E = 16 / (int)sizeof(IO), NW = NT / 32, U = 4;
  static_assert(RPC == 1 || NT == 32, "rows of a CTA share no barrier");
  __shared__ float s_m[NW], s_s[NW], s_cm[8], s_cs[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = RPC > 1 ? (int64_t)blockIdx.x * RPC + threadIdx.x / NT : blockIdx.x / C;
  const int tid = threadIdx.x % NT, lane = tid & 31, warp = tid >> 5;
  if (RPC > 1 && row >= a.rows) return;
  if (C > 1) cluster.barrier_arrive();  // waited for before another CTA's memory is touched
  const float c = ss::kLog2e / a.tau;
  const IO* x = (const IO*)a.logits + row * a.stride;
  const int lo = rank * a.split, n = a.V - lo < a.split ? (a.V - lo < 0 ? 0 : a.V - lo) : a.split;
  float m = -INFINITY, s = 0.f;
  auto raise = [&](float top) {
    if (top > m) {
      s *= ss::ex2((m - top) * c);
      m = top;
    }
  };
  // the first warp's first entries, their logits on the way while the row streams by
  float v0[2], x0[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int64_t t0 = -1;
    v0[i] = rank == 0 && warp == 0 && lane + 32 * i < a.K ? entry(a, row, lane + 32 * i, t0) : -INFINITY;
    x0[i] = v0[i] > -INFINITY ? ss::to_f(x[t0]) : 0.f;
  }
  const IO* xl = x + lo;
  const int head = head_of(xl, n), nv = (n - head) / E;
  for (int v = tid; v < nv; v += U * NT) {
    ss::Vec<IO, E> r[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < nv) r[i] = *reinterpret_cast<const ss::Vec<IO, E>*>(xl + head + (v + i * NT) * E);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < nv) top = fmaxf(top, vec_max(r[i]));
    raise(top);
    // with nothing above -inf so far only a NaN, which is no maximum, may reach the sum: 2^(c (-inf - 0)) is 0
    const ss::f2 base = ss::both(m > -INFINITY ? -m : 0.f), c2 = ss::both(c);
    ss::f2 p = 0;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < nv) {
#pragma unroll
        for (int e = 0; e < E; e += 2) p = ss::add2(p, ss::ex2_2(ss::mul2(ss::add2(ss::ld2(&r[i].v[e]), base), c2)));
      }
    const float2 q = ss::up(p);
    s += q.x + q.y;
  }
  for (int i = tid; i < n - nv * E; i += NT) {  // before and behind the vectors
    const float v = ss::to_f(xl[i < head ? i : i + nv * E]);
    raise(v);
    s += ss::ex2((m > -INFINITY ? v - m : v) * c);
  }
  // over the block, then the cluster; sums of empty parts weigh 2^-inf = 0
  auto join = [&](float m0, float s0, float m1) { return m0 > -INFINITY ? s0 * ss::ex2((m0 - m1) * c) : s0; };
  const float wm = warp_reduce(m, fmax_op), ws = warp_reduce(join(m, s, wm), add_op);
  float bm = wm, bs = ws;
  if (NW > 1) {
    if (lane == 0) s_m[warp] = wm, s_s[warp] = ws;
    __syncthreads();
    if (warp != 0 && C == 1) return;  // the first warp finishes the row: no further block barriers
    const float lm = lane < NW ? s_m[lane] : -INFINITY, lsum = lane < NW ? s_s[lane] : 0.f;
    bm = warp_reduce(lm, fmax_op), bs = warp_reduce(join(lm, lsum, bm), add_op);
  }
  if (C > 1) {
    cluster.barrier_wait();
    if (tid == 0) {
      *cluster.map_shared_rank(&s_cm[rank], 0) = bm;
      *cluster.map_shared_rank(&s_cs[rank], 0) = bs;
    }
    cluster.sync();
    if (rank != 0 || warp != 0) return;
    const float cm = lane < C ? s_cm[lane] : -INFINITY, cs = lane < C ? s_cs[lane] : 0.f;
    bm = warp_reduce(cm, fmax_op), bs = warp_reduce(join(cm, cs, bm), add_op);
  }
  const float ls = log2f(bs);
  // the teacher: maximum, sum, loss
  float top = fmaxf(v0[0], v0[1]);
  for (int k = lane + 64; k < a.K; k += 32) {
    int64_t t;
    top = fmaxf(top, entry(a, row, k, t));
  }
  top = warp_reduce(top, fmax_op);
  float sum = 0.f, dot = 0.f;  // dot: sum of weight x (log2 weight - log2 q)
  auto count = [&](float v, float xt) {
    const float w = weight(v, top, c);
    if (w > 0.f) {
      const float lw = v == top ? 0.f : (v - top) * c;
      sum += w;
      dot += w * (lw - ((xt - bm) * c - ls));
    }
  };
  count(v0[0], x0[0]);
  count(v0[1], x0[1]);
#pragma unroll 2
  for (int k = lane + 64; k < a.K; k += 32) {
    int64_t t;
    const float v = entry(a, row, k, t);
    if (v > -INFINITY) count(v, ss::to_f(x[t]));
  }
  sum = warp_reduce(sum, add_op);
  dot = warp_reduce(dot, add_op);
  if (lane == 0) {
    const bool some = top > -INFINITY;
    a.loss[row] = some ? a.tau * a.tau * 0.6931471805599453f * (dot / sum - log2f(sum)) : 0.f;
    a.valid[row] = some ? 1.f : 0.f;
    *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(bm, ls, top, some ? sum : 0.f);
  }
}

// grid rows x splits: every CTA its own part of a row. The sums over equal tokens: two bitmaps of
// the entries' low bits (seen, seen again) clear most of being repeated, and a warp looks together through all entries for
// each of the others (8192 x 32000, bf16: 172 us with 20 entries, 217 with 256, 399 with 1024; with every entry looking
// through all of them 172, 238 and 1500).
template <class IO, int NT, int RPC>
__global__ void __launch_bounds__(NT * RPC) k_distill_bwd(const DistillArgs a, int C) {
  static_assert(RPC == 1 || NT == 32, "rows of a CTA share no barrier");
  constexpr int E = 16 / (int)sizeof(IO), U = 4, KM = RPC > 1 ? kShortK : kMaxK, MARKS = RPC > 1 ? kShortV / 32 : kMarks;
  __shared__ float s_p_[RPC][KM];
  __shared__ int s_t_[RPC][KM];
  __shared__ unsigned s_seen_[RPC][MARKS], s_again_[RPC][MARKS];
  const int tid = threadIdx.x % NT, sub = threadIdx.x / NT;
  const int64_t row = RPC > 1 ? (int64_t)blockIdx.x * RPC + sub : blockIdx.x / C;
  if (RPC > 1 && row >= a.rows) return;
  const int rank = RPC > 1 ? 0 : (int)(blockIdx.x - row * C);
  float* s_p = s_p_[sub];
  int* s_t = s_t_[sub];
  unsigned *s_seen = s_seen_[sub], *s_again = s_again_[sub];
  auto sync = [] {
    if (RPC > 1) __syncwarp();
    else __syncthreads();
  };
  const int lo = rank * a.split, n = a.V - lo < a.split ? (a.V - lo < 0 ? 0 : a.V - lo) : a.split;
  const float4 st = *reinterpret_cast<const float4*>(a.stats + row * 4);
  const float c = ss::kLog2e / a.tau, g = a.dloss[row] * a.tau;
  const bool some = st.w > 0.f;
  const IO* x = (const IO*)a.logits + row * a.stride;
  IO* o = (IO*)a.dlogits + row * a.V;
  for (int i = tid; i < MARKS; i += NT) s_seen[i] = s_again[i] = 0;
  sync();
  for (int k = tid; k < a.K; k += NT) {
    int64_t t;
    const float v = entry(a, row, k, t);
    if (v > -INFINITY) {
      const unsigned w = (unsigned)t / 32 % MARKS, bit = 1u << (t & 31);
      if (atomicOr(&s_seen[w], bit) & bit) atomicOr(&s_again[w], bit);
    }
    s_t[k] = v > -INFINITY ? (int)t : -1;
    s_p[k] = v > -INFINITY ? weight(v, st.z, c) / st.w : 0.f;
  }
  auto grad = [&](float v) { return some ? g * ss::ex2(fmaf(v - st.x, c, -st.y)) : 0.f; };
  const IO* xl = x + lo;
  IO* ol = o + lo;
  // vectors where both rows reach 16 bytes at the same element
  const bool both = (((uintptr_t)xl ^ (uintptr_t)ol) & 15) == 0;
  const int head = both ? head_of(xl, n) : 0, nv = both ? (n - head) / E : 0;
#pragma unroll 1
  for (int v = tid; v < nv; v += U * NT) {
    ss::Vec<IO, E> r[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < nv) r[i] = *reinterpret_cast<const ss::Vec<IO, E>*>(xl + head + (v + i * NT) * E);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < nv) {
        ss::Vec<IO, E> y;
#pragma unroll
        for (int e = 0; e < E; e += 2)
          ss::st2(&y.v[e], ss::pk(grad(ss::to_f(r[i].v[e])), grad(ss::to_f(r[i].v[e + 1]))));
        *reinterpret_cast<ss::Vec<IO, E>*>(ol + head + (v + i * NT) * E) = y;
      }
  }
#pragma unroll 4
  for (int i = tid; i < n - nv * E; i += NT) {
    const int at = i < head ? i : i + nv * E;
    ss::from_f(ol[at], grad(ss::to_f(xl[at])));
  }
  sync();  // the entries' own values go over those above; equal tokens write the same sum
  const int lane = tid & 31;
  for (int k = tid; k - lane < a.K; k += NT) {
    const int t = k < a.K ? s_t[k] : -1;
    const bool mine = t >= lo && t < lo + n;
    float p = mine ? s_p[k] : 0.f;
    unsigned again = __ballot_sync(0xffffffffu, mine && s_again[(unsigned)t / 32 % MARKS] >> (t & 31) & 1);
    for (; again; again &= again - 1) {
      const int l = __ffs(again) - 1, tl = __shfl_sync(0xffffffffu, t, l);
      float q = 0.f;
      for (int j = lane; j < a.K; j += 32) q += s_t[j] == tl ? s_p[j] : 0.f;
      q = warp_reduce(q, add_op);
      if (lane == l) p = q;
    }
    if (!mine) continue;
    ss::from_f(o[t], g * (ss::ex2(fmaf(ss::to_f(x[t]) - st.x, c, -st.y)) - p));
  }
}

}  // namespace dst
}  // namespace atlas
