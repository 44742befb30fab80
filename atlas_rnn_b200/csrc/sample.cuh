// Token sampling: per row of logits, top-k, top-p and min-p filters on softmax(logits), then the argmax of
// logits / temperature plus Gumbel noise -log(-log u) from given uniforms (temperature <= 0: the argmax of the logits).
//
// Tokens are ordered by logit, ties by index (lowest first). A token's composite, (ordered bits of its logit) << 32 |
// ~index, makes that a total order, so each cut (top-k's last token, top-p's last token) is one composite.
// A token's mass is exp(logit - max) in units of 2^-40, an integer: sums of integers are the same in every
// order, so neither atomics nor the split over CTAs change a result.
//
// A row is shared by a cluster of 1 to 8 CTAs (more for few rows, where latency counts). Nothing of the row is kept on
// chip: the passes after the first read it from L2. The passes:
//   1. maximum and its index (the answer for a greedy row); per-thread maxima.
//   2. top-k up to kFastK: the k-th largest thread maximum bounds the k-th largest token from below, so a pass collects the
//      few tokens above that bound (a linear bin of 1/32 in the logit) into one CTA's list, which is sorted and finished
//      there: filters, noise of the survivors alone, argmax.
//   otherwise: a histogram over 2048 bins of (max - logit) * 32, counts or masses; the bin where the k-th token, or
//      the mass p, falls is collected and sorted if it holds at most kCap tokens (with all tokens above it, if those fit
//      too: then the list is finished as above), and else cut again by 11-bit digits of the composite.
//   3. with the cuts known and no complete list: a pass over the kept tokens for the argmax.
// Scores are compared in fp32; where two are closer than its error, in fp64, so the token is that of exact arithmetic.
// Bound: the logits once from HBM (the first pass) for large batches, the chain of passes and barriers for few rows.
#pragma once
#include <cooperative_groups.h>

#include "row_ops.cuh"

namespace atlas {
namespace smp {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kBins = 2048, kCap = 2048;
constexpr int kFastK = 512;
constexpr float kUnits = 1099511627776.f;  // 2^40

struct SampleArgs {
  const void* logits;  // [rows, V], rows `stride` elements apart
  const float* noise;  // [rows, V], `noise_stride` apart
  int64_t stride, noise_stride;
  int64_t* out;
  int V, split, vec;  // split: tokens per CTA, a multiple of 16
  // one setting for all rows, or one per row where the pointer is given
  double temperature, top_p, min_p;
  int64_t top_k;
  const float *temperature_row, *top_p_row, *min_p_row;
  const int* top_k_row;
};

struct Smem {
  unsigned cnt[kBins], lo[kBins], hi[kBins];  // this CTA's histogram: tokens, mass in two words
  unsigned tcnt[kBins];                       // the row's
  u64 tmass[kBins];
  u64 list[kCap];
  u64 wsum[32];
  unsigned wcnt[32];
  float wmax[32];
  int warg[32];
  double wscore[32];
  // per CTA of the cluster
  float cmax[8];
  int carg[8], cbin[8];
  double cscore[8];
  unsigned n;  // tokens collected (first CTA)
  // what a scan found: the bin, tokens and mass before it, its tokens; the row's totals
  int bin;
  unsigned before_n, in_n;
  u64 before_m, total_m;
  u64 cut;
};

__device__ __forceinline__ float clean(float l) { return l != l ? -INFINITY : l + 0.f; }  // NaN last; -0 is 0
__device__ __forceinline__ unsigned ordered(float l) {
  const unsigned b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 composite(float l, int i) { return (u64)ordered(l) << 32 | (unsigned)~i; }
__device__ __forceinline__ int index_of(u64 c) { return (int)~(unsigned)c; }
__device__ __forceinline__ float logit_of(u64 c) { return unordered((unsigned)(c >> 32)); }
// 32 bins a unit below the maximum; monotone in l, the maximum (infinite or not) in bin 0
__device__ __forceinline__ int linear_bin(float l, float m) {
  return l == m ? 0 : (int)fminf((m - l) * 32.f, (float)(kBins - 1));
}
__device__ __forceinline__ u64 mass(float l, float m) { return l == m ? (u64)kUnits : __float2ull_rn(expf(l - m) * kUnits); }

template <class T, class F>
__device__ __forceinline__ T warp_reduce(T v, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ void add_mass(Smem& s, int bin, u64 w) {
  const unsigned l = (unsigned)w, old = atomicAdd(&s.lo[bin], l);
  const unsigned h = (unsigned)(w >> 32) + (old + l < old);
  if (h) atomicAdd(&s.hi[bin], h);
}

// Exact score of a token, in fp64.
__device__ __forceinline__ double score64(float l, float u, double temperature) {
  const double e = -log(fmax((double)u, 1e-20));
  return (double)l / temperature - log(fmax(e, 1e-20));
}

// A thread's best token so far. Scores closer than the fp32 error are settled in fp64; equal ones by index.
struct Best {
  float score = -INFINITY, l = 0.f, u = 0.f;
  int i = 0x7fffffff;
  __device__ __forceinline__ static float margin(float s) { return 2e-5f + 1e-6f * fabsf(s); }
  __device__ __forceinline__ void offer(float l2, float u2, int i2, float inv_t, double temperature) {
    const float a = l2 == INFINITY ? l2 : l2 * inv_t;
    const bool none = i == 0x7fffffff;
    // -log u >= 1 - u: a token with 1 - u above exp(a - score) stays below the best (1e-3: the roundings here)
    if (!none && 1.f - u2 > ss::ex2((a - score + 1e-3f) * ss::kLog2e)) return;
    const float s = a - logf(fmaxf(-logf(fmaxf(u2, 1e-20f)), 1e-20f));
    bool better = none || s > score;
    if (!none && !(fabsf(s - score) > margin(s))) {  // too close, or beyond fp32
      const double x = score64(l2, u2, temperature), y = score64(l, u, temperature);
      better = x > y || (x == y && i2 < i);
    }
    if (better) score = s, l = l2, u = u2, i = i2;
  }
};

template <class IO, int NT>
struct Row {
  const IO* p;
  const float* noise;
  int lo, n, vec, tid;
  // f(index, logit) over the CTA's tokens that are not masked out, a thread's in ascending order
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int E = 16 / (int)sizeof(IO);
    int done = 0;
    if (vec) {
      const int nv = n / E;
#pragma unroll 4
      for (int v = tid; v < nv; v += NT) {
        const ss::Vec<IO, E> x = *reinterpret_cast<const ss::Vec<IO, E>*>(p + lo + v * E);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float l = clean(ss::to_f(x.v[e]));
          if (l > -INFINITY) f(lo + v * E + e, l);
        }
      }
      done = nv * E;
    }
    for (int k = done + tid; k < n; k += NT) {
      const float l = clean(ss::to_f(p[lo + k]));
      if (l > -INFINITY) f(lo + k, l);
    }
  }
};

// Reads of another CTA's shared memory end at a cluster barrier before that CTA may leave: every path does the same barriers.
template <class IO, int NT>
__global__ void __launch_bounds__(NT) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char sm_raw[];
  Smem& s = *reinterpret_cast<Smem*>(sm_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NW = NT / 32;
  cluster.barrier_arrive();  // waited for before the first access to another CTA's memory: it has to have started
  Smem& first = *cluster.map_shared_rank(&s, 0);

  const double temperature = fmin(a.temperature_row ? (double)a.temperature_row[row] : a.temperature, 1e300);
  const double top_p = a.top_p_row ? (double)a.top_p_row[row] : a.top_p;
  const double min_p = a.min_p_row ? (double)a.min_p_row[row] : a.min_p;
  int64_t k = a.top_k_row ? a.top_k_row[row] : a.top_k;
  if (!(top_p > 0.0) || !(min_p <= 1.0) || !(temperature > 0.0)) k = 1;  // nothing but the first token
  const bool need_k = k >= 1 && k < a.V, need_p = top_p < 1.0;
  const float inv_t = (float)fmin(1.0 / temperature, 1e30);  // beyond: settled in fp64 by Best

  Row<IO, NT> r;
  r.p = (const IO*)a.logits + row * a.stride;
  r.noise = a.noise + row * a.noise_stride;
  r.lo = rank * a.split;
  r.n = a.V - r.lo < a.split ? (a.V - r.lo < 0 ? 0 : a.V - r.lo) : a.split;
  r.vec = a.vec, r.tid = tid;

  // ---- maximum, its lowest index
  float tmax = -INFINITY;
  int targ = 0x7fffffff;
  r.each([&](int i, float l) {
    if (l > tmax) tmax = l, targ = i;
  });
  {
    const float wm = warp_reduce(tmax, [](float x, float y) { return fmaxf(x, y); });
    const int wa = warp_reduce(tmax == wm ? targ : 0x7fffffff, [](int x, int y) { return min(x, y); });
    if (lane == 0) s.wmax[warp] = wm, s.warg[warp] = wa;
    if (tid == 0) s.n = 0;
    __syncthreads();
    cluster.barrier_wait();
    if (warp == 0) {
      const float x = lane < NW ? s.wmax[lane] : -INFINITY;
      const float bm = warp_reduce(x, [](float p, float q) { return fmaxf(p, q); });
      const int ba = warp_reduce(lane < NW && x == bm ? s.warg[lane] : 0x7fffffff, [](int p, int q) { return min(p, q); });
      if (lane < C) {
        Smem& o = *cluster.map_shared_rank(&s, lane);
        o.cmax[rank] = bm;
        o.carg[rank] = ba;
      }
    }
    cluster.sync();
  }
  float m = s.cmax[0];
  for (int c = 1; c < C; ++c) m = fmaxf(m, s.cmax[c]);
  if (!(m > -INFINITY) || k == 1) {  // nothing to draw from, or the first token alone
    if (rank == 0 && tid == 0) {
      int best = 0x7fffffff;
      for (int c = 0; c < C; ++c)
        if (s.cmax[c] == m) best = min(best, s.carg[c]);
      a.out[row] = m > -INFINITY ? best : 0;
    }
    return;  // the same for the whole cluster
  }
  // w >= min_p as a bound on the logit: the smallest float at or above max + log(min_p)
  const float floor_l = min_p > 0.0 ? __double2float_ru((double)m + log(min_p)) : -INFINITY;

  // Exclusive prefix of (count, mass) over the row's bins; finds the bin where `target` falls: before < target <=
  // before + its own (by mass or by count). s.bin = -1 where the row ends first.
  auto find = [&](bool by_mass, u64 target) {
    constexpr int PER = kBins / NT;
    unsigned c[PER];
    u64 w[PER], cs = 0, ws = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = s.tcnt[tid * PER + i];
      w[i] = by_mass ? s.tmass[tid * PER + i] : c[i];
      cs += c[i], ws += w[i];
    }
    u64 pc = cs, pw = ws;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, pc, o), y = __shfl_up_sync(0xffffffffu, pw, o);
      if (lane >= o) pc += x, pw += y;
    }
    if (lane == 31) s.wcnt[warp] = (unsigned)pc, s.wsum[warp] = pw;
    if (tid == 0) s.bin = -1;
    __syncthreads();
    u64 bc = pc - cs, bw = pw - ws;
    for (int i = 0; i < warp; ++i) bc += s.wcnt[i], bw += s.wsum[i];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (bw < target && target <= bw + w[i]) {
        s.bin = tid * PER + i;
        s.before_n = (unsigned)bc, s.in_n = c[i], s.before_m = bw;
      }
      bc += c[i], bw += w[i];
    }
    if (tid == NT - 1) s.total_m = bw;
    __syncthreads();
  };
  // The CTAs' histograms added: each adds a share of the bins and hands it to all.
  auto share = [&](bool by_mass) {
    cluster.sync();
    const int per = kBins / C;
    for (int i = tid; i < per; i += NT) {
      const int bin = rank * per + i;
      unsigned c = 0;
      u64 w = 0;
      for (int q = 0; q < C; ++q) {
        const Smem& o = *cluster.map_shared_rank(&s, q);
        c += o.cnt[bin];
        if (by_mass) w += (u64)o.hi[bin] << 32, w += o.lo[bin];
      }
      for (int q = 0; q < C; ++q) {
        Smem& o = *cluster.map_shared_rank(&s, q);
        o.tcnt[bin] = c;
        if (by_mass) o.tmass[bin] = w;
      }
    }
    cluster.sync();
  };
  auto clear = [&] {
    for (int i = tid; i < kBins; i += NT) s.cnt[i] = s.lo[i] = s.hi[i] = 0;
    __syncthreads();
  };
  // A token into the first CTA's list.
  auto push = [&](u64 c) {
    const unsigned at = atomicAdd(&first.n, 1u);
    if (at < kCap) first.list[at] = c;
  };
  // The first CTA's list in descending order (bitonic over the next power of two).
  auto sort = [&](int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += NT) s.list[i] = 0;
    __syncthreads();
    for (int w = 2; w <= size; w <<= 1)
      for (int d = w >> 1; d > 0; d >>= 1) {
        for (int i = tid; i < size / 2; i += NT) {
          const int x = i / d * 2 * d + i % d, y = x + d;
          const u64 p = s.list[x], q = s.list[y];
          if ((p < q) == ((x & w) == 0)) s.list[x] = q, s.list[y] = p;
        }
        __syncthreads();
      }
  };
  // Inclusive-to-exclusive prefix of the list's masses (each of `n` entries, strided by thread blocks of PER).
  constexpr int LP = kCap / NT;
  auto list_prefix = [&](int n, u64 (&before)[LP], u64 (&own)[LP], u64& total) {
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < LP; ++i) {
      const int at = tid * LP + i;
      own[i] = at < n ? mass(logit_of(s.list[at]), m) : 0;
      sum += own[i];
    }
    u64 inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s.wsum[warp] = inc;
    __syncthreads();
    u64 b = inc - sum;
    total = 0;
    for (int i = 0; i < NW; ++i) {
      if (i < warp) b += s.wsum[i];
      total += s.wsum[i];
    }
#pragma unroll
    for (int i = 0; i < LP; ++i) before[i] = b, b += own[i];
    __syncthreads();
  };
  // The CTA's best token: fp32 scores, the ones within its error of the best again in fp64.
  auto block_best = [&](const Best& b, double& score, int& index) {
    const float wm = warp_reduce(b.score, [](float x, float y) { return fmaxf(x, y); });
    if (lane == 0) s.wmax[warp] = wm;
    __syncthreads();
    float top = s.wmax[0];
    for (int i = 1; i < NW; ++i) top = fmaxf(top, s.wmax[i]);
    const bool near = b.i != 0x7fffffff && (b.score == top || b.score >= top - 2.f * Best::margin(top));
    double x = near ? score64(b.l, b.u, temperature) : -INFINITY;
    int at = near ? b.i : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double y = __shfl_xor_sync(0xffffffffu, x, o);
      const int i = __shfl_xor_sync(0xffffffffu, at, o);
      if (y > x || (y == x && i < at)) x = y, at = i;
    }
    if (lane == 0) s.wscore[warp] = x, s.warg[warp] = at;
    __syncthreads();
    score = -INFINITY, index = 0x7fffffff;
    for (int i = 0; i < NW; ++i)
      if (s.wscore[i] > score || (s.wscore[i] == score && s.warg[i] < index)) score = s.wscore[i], index = s.warg[i];
  };
  auto cut_at = [&](u64 total) { return (u64)ceil(top_p * (double)total); };  // kept while the mass before is below
  // The first CTA's list holds every token down to the last kept one: its filters, its draw. total: the mass that top-p
  // is a share of, 0 for the list's own (after top-k).
  auto finish = [&](int n, u64 total) {
    sort(n);
    if (need_k && k < n) n = (int)k;
    u64 before[LP], own[LP], sum;
    list_prefix(n, before, own, sum);
    const u64 cut = need_p ? cut_at(total ? total : sum) : ~0ull;
    Best b;
#pragma unroll
    for (int i = 0; i < LP; ++i) {
      const int at = tid * LP + i;
      if (at >= n || !(at == 0 || before[i] < cut)) continue;
      const u64 c = s.list[at];
      const float l = logit_of(c);
      if (l >= floor_l) b.offer(l, r.noise[index_of(c)], index_of(c), inv_t, temperature);
    }
    double score;
    int index;
    block_best(b, score, index);
    if (tid == 0) a.out[row] = index;
  };

  u64 keep = 0;  // tokens with a composite below are cut
  // ---- top-k through the thread maxima
  if (need_k && k <= kFastK && k <= NT) {
    clear();
    if (tmax > -INFINITY) atomicAdd(&s.cnt[linear_bin(tmax, m)], 1u);
    __syncthreads();
    for (int i = tid; i < kBins; i += NT) s.tcnt[i] = s.cnt[i];
    __syncthreads();
    find(false, (u64)k);
    if (tid < C) cluster.map_shared_rank(&s, tid)->cbin[rank] = s.bin < 0 ? kBins - 1 : s.bin;
    cluster.sync();
    int bound = s.cbin[0];  // k thread maxima of one CTA lie in bins up to its bound
    for (int c = 1; c < C; ++c) bound = min(bound, s.cbin[c]);
    r.each([&](int i, float l) {
      if (linear_bin(l, m) <= bound) push(composite(l, i));
    });
    cluster.sync();
    const unsigned n = first.n;
    cluster.sync();
    if (n <= kCap) {
      if (rank == 0) finish((int)n, 0);
      return;
    }
    if (rank == 0 && tid == 0) s.n = 0;  // too many: the general cut below, whose barriers come before its first push
  }

  // ---- one cut: the last token with fewer than `target` tokens (less than `target` of mass) before it, among those from
  // `keep` on; true where that finished the row.
  auto descend = [&](bool by_mass) {
    u64 target = by_mass ? 0 : (u64)k, total = 0, before = 0, prefix = 0;
    // the group of tokens that is being cut: linear bin `lin` (-1: all), composite >> shift == prefix
    int lin = -1, shift = 64;
    for (;;) {
      const int low = shift > 11 ? shift - 11 : 0, last = (1 << (shift - low)) - 1;
      auto bin_of = [&](u64 c, float l) {  // -1: outside the group
        const int b = linear_bin(l, m);
        if (lin < 0) return c < keep ? -1 : b;
        if (c < keep || b != lin || (shift < 64 && (c >> shift) != prefix)) return -1;
        return last - ((int)(c >> low) & last);
      };
      clear();
      r.each([&](int i, float l) {
        const int b = bin_of(composite(l, i), l);
        if (b < 0) return;
        atomicAdd(&s.cnt[b], 1u);
        if (by_mass) add_mass(s, b, mass(l, m));
      });
      share(by_mass);
      if (lin < 0 && by_mass) {
        find(true, ~0ull);
        total = s.total_m;
        target = cut_at(total);
      }
      find(by_mass, target - before);
      const int bin = s.bin;
      if (bin < 0) return false;  // every token is kept
      const bool all = lin < 0 && s.before_n + s.in_n <= kCap;  // with all tokens above it
      if (all || s.in_n <= kCap) {
        r.each([&](int i, float l) {
          const u64 c = composite(l, i);
          const int b = bin_of(c, l);
          if (b == bin || (all && b >= 0 && b < bin)) push(c);
        });
        cluster.sync();
        const int n = (int)first.n;
        cluster.sync();
        if (all) {
          if (rank == 0) finish(n, total);
          return true;
        }
        if (rank == 0) {
          sort(n);
          const u64 t = target - before - s.before_m;  // within the bin
          if (by_mass) {
            u64 b[LP], own[LP], sum;
            list_prefix(n, b, own, sum);
#pragma unroll
            for (int j = 0; j < LP; ++j)
              if (tid * LP + j < n && b[j] < t && (tid * LP + j == n - 1 || b[j] + own[j] >= t)) s.cut = s.list[tid * LP + j];
          } else if (tid == 0) {
            s.cut = s.list[t - 1];
          }
          if (tid == 0) s.n = 0;
          __syncthreads();
          const u64 cut = s.cut;
          if (tid < C) cluster.map_shared_rank(&s, tid)->cut = cut;
        }
        cluster.sync();
        keep = s.cut;
        return false;
      }
      before += s.before_m;
      if (lin < 0) {
        lin = bin;
      } else {
        prefix = shift < 64 ? prefix << (shift - low) | (u64)(last - bin) : (u64)(last - bin);
        shift = low;
      }
      __syncthreads();
    }
  };
  if (need_k && descend(false)) return;
  if (need_p && descend(true)) return;

  // ---- the kept tokens' argmax
  Best b;
  r.each([&](int i, float l) {
    if (l >= floor_l && composite(l, i) >= keep) b.offer(l, r.noise[i], i, inv_t, temperature);
  });
  double score;
  int index;
  block_best(b, score, index);
  if (tid == 0) first.cscore[rank] = score, first.carg[rank] = index;
  cluster.sync();
  if (rank == 0 && tid == 0) {
    for (int c = 0; c < C; ++c)
      if (s.cscore[c] > score || (s.cscore[c] == score && s.carg[c] < index)) score = s.cscore[c], index = s.carg[c];
    a.out[row] = index;
  }
}

}  // namespace smp
}  // namespace atlas
