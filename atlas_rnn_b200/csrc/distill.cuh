// Distillation from a teacher's top logits, forward and backward. Per row, with the teacher's entries (value v_k, token i_k;
// entries with i_k outside 0 .. V-1, or -inf or NaN values, are absent) and the student's logits x:
//   p = softmax(v / tau) over the entries,  q = softmax(x / tau) over the vocabulary,
//   loss = tau^2 sum_k p_k (log p_k - log q_{i_k}),   d loss / d x_j = tau (q_j - sum_{k: i_k = j} p_k)
// (tokens may repeat), and 0 for a row without entries. The forward reads the logits once with a running maximum m and
// sum s = sum 2^(c (x - m)), c = log2(e) / tau, so log2 q_j = c (x_j - m) - log2 s; the difference is taken first, so that
// logits of any size keep their distances. The backward reads them again, writes tau g q everywhere, and then the
// entries' own values.
// HBM-bound: 3 x rows x V elements over both. Few rows are split over a cluster of CTAs.
#pragma once
#include <cooperative_groups.h>

#include "row_ops.cuh"

namespace atlas {
namespace dst {

namespace cg = cooperative_groups;
constexpr int kMaxK = 1024;

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
  int V, K, split, vec;
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

// grid rows x cluster
template <class IO, int NT>
__global__ void __launch_bounds__(NT) k_distill_fwd(const DistillArgs a) {
  constexpr int E = 16 / (int)sizeof(IO), NW = NT / 32, U = 4;
  __shared__ float s_m[NW], s_s[NW], s_cm[8], s_cs[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
  int done = 0;
  if (a.vec) {
    const int nv = n / E;
    int v = tid;
    for (; v + (U - 1) * NT < nv; v += U * NT) {
      ss::Vec<IO, E> r[U];
#pragma unroll
      for (int i = 0; i < U; ++i) r[i] = *reinterpret_cast<const ss::Vec<IO, E>*>(x + lo + (v + i * NT) * E);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, ss::to_f(r[i].v[e]));
      raise(top);
      if (m > -INFINITY) {
        float p[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) p[e & 1] += ss::ex2((ss::to_f(r[i].v[e]) - m) * c);
        s += p[0] + p[1];
      }
    }
    for (; v < nv; v += NT) {
      const ss::Vec<IO, E> r = *reinterpret_cast<const ss::Vec<IO, E>*>(x + lo + v * E);
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < E; ++e) top = fmaxf(top, ss::to_f(r.v[e]));
      raise(top);
      if (m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < E; ++e) s += ss::ex2((ss::to_f(r.v[e]) - m) * c);
      }
    }
    done = nv * E;
  }
  for (int i = done + tid; i < n; i += NT) {
    const float v = ss::to_f(x[lo + i]);
    raise(v);
    if (m > -INFINITY) s += ss::ex2((v - m) * c);
    else if (v != v) s = v;  // a NaN is no maximum: it has to reach the sum
  }
  // over the block, then the cluster; sums of empty parts weigh 2^-inf = 0
  auto join = [&](float m0, float s0, float m1) { return m0 > -INFINITY ? s0 * ss::ex2((m0 - m1) * c) : s0; };
  float wm = warp_reduce(m, fmax_op);
  float ws = warp_reduce(join(m, s, wm), add_op);
  if (lane == 0) s_m[warp] = wm, s_s[warp] = ws;
  __syncthreads();
  float bm = s_m[0], bs = 0.f;
  for (int i = 1; i < NW; ++i) bm = fmaxf(bm, s_m[i]);
  for (int i = 0; i < NW; ++i) bs += join(s_m[i], s_s[i], bm);
  if (C > 1) {
    cluster.barrier_wait();
    if (tid == 0) {
      *cluster.map_shared_rank(&s_cm[rank], 0) = bm;
      *cluster.map_shared_rank(&s_cs[rank], 0) = bs;
    }
    cluster.sync();
    if (rank != 0) return;
    bm = s_cm[0], bs = 0.f;
    for (int i = 1; i < C; ++i) bm = fmaxf(bm, s_cm[i]);
    for (int i = 0; i < C; ++i) bs += join(s_cm[i], s_cs[i], bm);
  }
  const float ls = log2f(bs);
  // the teacher: maximum, sum, loss
  float top = -INFINITY;
  for (int k = tid; k < a.K; k += NT) {
    int64_t t;
    top = fmaxf(top, entry(a, row, k, t));
  }
  top = warp_reduce(top, fmax_op);
  __syncthreads();
  if (lane == 0) s_m[warp] = top;
  __syncthreads();
  for (int i = 0; i < NW; ++i) top = fmaxf(top, s_m[i]);
  float sum = 0.f, dot = 0.f;  // dot: sum of weight x (log2 weight - log2 q)
  for (int k = tid; k < a.K; k += NT) {
    int64_t t;
    const float v = entry(a, row, k, t), w = weight(v, top, c);
    if (w > 0.f) {
      const float lw = v == top ? 0.f : (v - top) * c;
      sum += w;
      dot += w * (lw - ((ss::to_f(x[t]) - bm) * c - ls));
    }
  }
  sum = warp_reduce(sum, add_op);
  dot = warp_reduce(dot, add_op);
  __syncthreads();
  if (lane == 0) s_m[warp] = sum, s_s[warp] = dot;
  __syncthreads();
  if (tid == 0) {
    sum = dot = 0.f;
    for (int i = 0; i < NW; ++i) sum += s_m[i], dot += s_s[i];
    const bool some = top > -INFINITY;
    a.loss[row] = some ? a.tau * a.tau * 0.6931471805599453f * (dot / sum - log2f(sum)) : 0.f;
    a.valid[row] = some ? 1.f : 0.f;
    *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(bm, ls, top, some ? sum : 0.f);
  }
}

// grid (splits, rows): every CTA its own part of a row
template <class IO, int NT>
__global__ void __launch_bounds__(NT) k_distill_bwd(const DistillArgs a, int C) {
  constexpr int E = 16 / (int)sizeof(IO), U = 4;
  __shared__ float s_p[kMaxK];
  __shared__ int s_t[kMaxK];
  const int64_t row = blockIdx.x / C;
  const int rank = (int)(blockIdx.x - row * C), tid = threadIdx.x;
  const int lo = rank * a.split, n = a.V - lo < a.split ? (a.V - lo < 0 ? 0 : a.V - lo) : a.split;
  const float4 st = *reinterpret_cast<const float4*>(a.stats + row * 4);
  const float c = ss::kLog2e / a.tau, g = a.dloss[row] * a.tau;
  const bool some = st.w > 0.f;
  const IO* x = (const IO*)a.logits + row * a.stride;
  IO* o = (IO*)a.dlogits + row * a.V;
  for (int k = tid; k < a.K; k += NT) {
    int64_t t;
    const float v = entry(a, row, k, t);
    s_t[k] = v > -INFINITY ? (int)t : -1;
    s_p[k] = v > -INFINITY ? weight(v, st.z, c) / st.w : 0.f;
  }
  auto grad = [&](float v) { return some ? g * ss::ex2(fmaf(v - st.x, c, -st.y)) : 0.f; };
  int done = 0;
  if (a.vec) {
    const int nv = n / E;
#pragma unroll 1
    for (int v = tid; v < nv; v += U * NT) {
      ss::Vec<IO, E> r[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (v + i * NT < nv) r[i] = *reinterpret_cast<const ss::Vec<IO, E>*>(x + lo + (v + i * NT) * E);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (v + i * NT < nv) {
          ss::Vec<IO, E> y;
#pragma unroll
          for (int e = 0; e < E; e += 2)
            ss::st2(&y.v[e], ss::pk(grad(ss::to_f(r[i].v[e])), grad(ss::to_f(r[i].v[e + 1]))));
          *reinterpret_cast<ss::Vec<IO, E>*>(o + lo + (v + i * NT) * E) = y;
        }
    }
    done = nv * E;
  }
  for (int i = done + tid; i < n; i += NT) ss::from_f(o[lo + i], grad(ss::to_f(x[lo + i])));
  __syncthreads();  // the entries' own values go over those above; equal tokens write the same sum
  for (int k = tid; k < a.K; k += NT) {
    const int t = s_t[k];
    if (t < lo || t >= lo + n) continue;
    float p = 0.f;
    for (int j = 0; j < a.K; ++j) p += s_t[j] == t ? s_p[j] : 0.f;
    ss::from_f(o[t], g * (ss::ex2(fmaf(ss::to_f(x[t]) - st.x, c, -st.y)) - p));
  }
}

}  // namespace dst
}  // namespace atlas
