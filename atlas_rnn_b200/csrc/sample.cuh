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
//   1. the maximum (a greedy row: and its lowest index, done); per-thread maxima.
//   2. top-k up to kFastK: the k-th largest thread maximum bounds the k-th largest token from below, so a pass collects the
//      few tokens above that bound (to 1/64 in the logit) into one CTA's list, which is sorted and finished
//      there: filters, noise of the survivors alone, argmax.
//   otherwise: a histogram over 2048 bins of (max - logit) * 64, counts or masses; the bin where the k-th token, or
//      the mass p, falls is collected and sorted if it holds at most kCap tokens (with all tokens above it, if those fit
//      too: then the list is finished as above), and else cut again by 11-bit digits of the composite.
//   3. with the cuts known and no complete list: a pass over the kept tokens for the argmax.
// Scores are compared in fp32; where two are closer than its error, in fp64, so the token is that of exact arithmetic.
// Masses are added as two 32-bit words with a carry: a 64-bit atomic on shared memory is emulated (65536 of them a CTA
// over 256 bins took 49 us, the two words 12).
// Bound: the logits once from HBM (the first pass) for large batches, the chain of passes and barriers for few rows (bf16
// rows of 131072: 1 greedy row 5 us, with top-k 50 15; 64 rows 9 greedy, 22 with top-k 50, 32 with min-p alone, 80 with
// top-p alone, whose histogram and final pass go over most of the tokens).
#pragma once
#include <cfloat>
#include <cooperative_groups.h>

#include "row_ops.cuh"

namespace atlas {
namespace smp {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kBins = 2048, kCap = 2048;
constexpr int kFastK = 512;
constexpr int kNone = 0x7fffffff;
constexpr int kMaxV = (1 << 24) - 16;  // as many masses of up to 2^40 add up to less than 2^64

struct SampleArgs {
  const void* logits;  // [rows, V], rows `stride` elements apart
  const float* noise;  // [rows, V], `noise_stride` apart
  int64_t stride, noise_stride;
  int64_t* out;
  int V, split;  // split: tokens per CTA, a multiple of 16
  // one setting for all rows, or one per row where the pointer is given
  double temperature, top_p, min_p;
  int64_t top_k;
  const float *temperature_row, *top_p_row, *min_p_row;
  const int* top_k_row;
};

struct alignas(16) Smem {
  unsigned lo[kBins], hi[kBins];  // this CTA's histogram: counts, or masses in two words
  u64 sum[kBins];                 // the row's
  u64 list[kCap];                 // (first CTA) the row's collected tokens
  u64 mine[kCap];                 // this CTA's
  u64 wsum[32];
  float west[32], wmax[32];
  int warg[32];
  double wscore[32];
  // per CTA of the cluster
  float cmax[8];
  int carg[8], cbin[8];
  double cscore[8];
  unsigned n, n_mine, base;  // tokens collected: the row's (first CTA), this CTA's; its place among them
  // what find() found: the bin, the weight before it, about how many tokens before and in it
  int bin;
  float est_before, est_in;
  u64 before, cut;
};

__device__ __forceinline__ float clean(float l) { return l > -INFINITY ? l + 0.f : -INFINITY; }  // NaN last; -0 is 0
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
// 64 bins a unit below the (finite) maximum, to the nearest; monotone in l
__device__ __forceinline__ int linear_bin(float l, float m) {
  return __float_as_int(fminf((m - l) * 64.f, (float)(kBins - 1)) + 8388608.f) & (kBins - 1);
}
// exp(l - m) in units of 2^-40, rounded down: the 24 bits of the fp32 value, shifted; in two words. Off by at most (d + 1) 2^-22
// of itself at d = m - l (three roundings of the exponent, 3 d 2^-24, and the hardware's exp2, 2^-22): at most 2^-21 of the largest.
__device__ __forceinline__ uint2 mass2(float l, float m) {
  const unsigned b = __float_as_uint(ss::ex2((l - m) * ss::kLog2e));
  const int sh = (int)(b >> 23) - 110;  // at most 17
  const unsigned f = (b & 0x7fffffu) | 0x800000u;
  unsigned up, down, hi;  // shifts of 32 and more (also negative ones, as unsigned) give 0
  asm("shl.b32 %0, %1, %2;" : "=r"(up) : "r"(f), "r"(sh));
  asm("shr.u32 %0, %1, %2;" : "=r"(down) : "r"(f), "r"(-sh));
  asm("shr.u32 %0, %1, %2;" : "=r"(hi) : "r"(f), "r"(32 - sh));
  return make_uint2(sh >= 0 ? up : down, hi);
}
__device__ __forceinline__ u64 mass(float l, float m) {
  const uint2 w = mass2(l, m);
  return (u64)w.y << 32 | w.x;
}

template <class T, class F>
__device__ __forceinline__ T warp_reduce(T v, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <class T>
__device__ __forceinline__ T warp_scan(T v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}
__device__ __forceinline__ float fmax_op(float x, float y) { return fmaxf(x, y); }
__device__ __forceinline__ int imin_op(int x, int y) { return min(x, y); }

// Exact score of a token, in fp64. A call: inlined at its five places it made the kernel too long for the others.
__device__ __noinline__ double score64(float l, float u, double temperature) {
  const double e = -log(fmax((double)u, 1e-20));
  return (double)l / temperature - log(fmax(e, 1e-20));
}

// A token's score in fp32: e = -log u by the hardware's log2 (absolute error 2^-22, so 1.7e-5 of e down to u = 0.99),
// above that by its series in 1 - u; -log e by it too (2^-22 of at most 66): 4e-5 in all, and the rounding of l / temperature.
__device__ __forceinline__ float score32(float l, float u, float inv_t) {
  const float t = 1.f - u, e0 = -0.6931471805599453f * ss::lg2(fmaxf(u, 1e-20f));
  const float e = fmaxf(t < 0.01f ? t * fmaf(t, fmaf(t, 1.f / 3.f, 0.5f), 1.f) : e0, 1e-20f);
  return fmaf(-0.6931471805599453f, ss::lg2(e), l * inv_t);
}
__device__ __forceinline__ float margin(float s) { return 2e-4f + 2e-6f * fabsf(s); }

// A thread's best token so far; scores closer than their error are settled in fp64, equal ones by index.
struct Best {
  float score = -INFINITY, l = 0.f, u = 0.f;
  int i = kNone;
  __device__ __forceinline__ void offer(float s, float l2, float u2, int i2, double temperature) {
    bool better = i == kNone || s > score;
    if (i != kNone && !(fabsf(s - score) > margin(s))) {
      const double x = score64(l2, u2, temperature), y = score64(l, u, temperature);
      better = x > y || (x == y && i2 < i);
    }
    if (better) score = s, l = l2, u = u2, i = i2;
  }
};

constexpr int kBatch = 8;  // tokens a thread works on at a time, independent of one another
constexpr int kAhead = 6;  // batches on their way from L2 meanwhile (one: a pass over 65536 tokens a CTA took 10 us, not 5)
template <class IO, int NT>
struct Row {
  static constexpr int E = 16 / (int)sizeof(IO), U = kBatch / E;
  struct Ring {
    uint4 v[kAhead + 1][U][NT];
  };
  const IO* p;
  Ring* ring;
  int lo, n, tid;
  // f(logits, indices) over the CTA's tokens in batches; a logit as it is in memory, NaN in the places that are none. Each
  // thread feeds itself through its own slots of the ring.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    float l[kBatch];
    int id[kBatch];
    // vectors from the row's first 16-byte boundary on
    const IO* q0 = p + lo;
    int head = (int)((16 - ((uintptr_t)q0 & 15)) & 15) / (int)sizeof(IO);
    head = head < n ? head : n;
    const int nv = (n - head) / E;
    int next = tid, put = 0, get = 0;
    auto load = [&] {
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (next + q * NT < nv) ss::cp_piece<16>(&ring->v[put][q][tid], q0 + head + (next + q * NT) * E, 16);
      ss::cp_commit();
      next += U * NT;
      put = put == kAhead ? 0 : put + 1;
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load();
    int v = tid, k = tid;  // next vector, next single token beside the vectors
#pragma unroll 1
    for (;;) {
      if (v < nv) {
        ss::cp_wait<kAhead - 1>();
#pragma unroll
        for (int q = 0; q < U; ++q) {
          const uint4 raw = ring->v[get][q][tid];
          const ss::Vec<IO, E> x = *reinterpret_cast<const ss::Vec<IO, E>*>(&raw);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            id[q * E + e] = lo + head + (v + q * NT) * E + e;
            l[q * E + e] = v + q * NT < nv ? ss::to_f(x.v[e]) : NAN;
          }
        }
        v += U * NT;
        get = get == kAhead ? 0 : get + 1;
        load();  // into the slot of the batch before this one
      } else if (k < n - nv * E) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const int at = k + e * NT;
          id[e] = lo + (at < head ? at : at + nv * E);
          l[e] = at < n - nv * E ? ss::to_f(p[id[e]]) : NAN;
        }
        k += kBatch * NT;
      } else {
        break;
      }
      f(l, id);  // in one place: it is inlined, and the batch stays in registers
    }
    ss::cp_wait<0>();
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

  Row<IO, NT> r;
  r.p = (const IO*)a.logits + row * a.stride;
  r.lo = rank * a.split;
  r.n = a.V - r.lo < a.split ? (a.V - r.lo < 0 ? 0 : a.V - r.lo) : a.split;
  r.tid = tid;
  r.ring = reinterpret_cast<typename Row<IO, NT>::Ring*>(sm_raw + sizeof(Smem));
  const float* noise = a.noise + row * a.noise_stride;

  const double t_given = a.temperature_row ? (double)a.temperature_row[row] : a.temperature;
  const double temperature = fmin(t_given, 1e300);  // a NaN becomes 1e300: it is caught before
  const double top_p = a.top_p_row ? (double)a.top_p_row[row] : a.top_p;
  const double min_p = a.min_p_row ? (double)a.min_p_row[row] : a.min_p;
  int64_t k = a.top_k_row ? a.top_k_row[row] : a.top_k;
  if (!(top_p > 0.0) || !(min_p <= 1.0) || !(t_given >= 1e-30)) k = 1;  // nothing but the first token (NaNs too)
  const bool need_k = k >= 1 && k < a.V, need_p = top_p < 1.0;
  const float inv_t = (float)(1.0 / fmax(temperature, 1e-30));

  auto block_max = [&](float v) {
    const float wm = warp_reduce(v, fmax_op);
    if (lane == 0) s.wmax[warp] = wm;
    __syncthreads();
    return warp_reduce(lane < NW ? s.wmax[lane] : -INFINITY, fmax_op);
  };

  // ---- maximum
  float tmax = -INFINITY;  // the thread's largest logit (a NaN is none)
  r.each([&](const float(&l)[kBatch], const int(&)[kBatch]) {
#pragma unroll
    for (int e = 0; e < kBatch; ++e) tmax = fmaxf(tmax, l[e]);
  });
  {
    const float bm = block_max(tmax);
    if (tid == 0) s.n = s.n_mine = 0;
    cluster.barrier_wait();
    if (tid < C) cluster.map_shared_rank(&s, tid)->cmax[rank] = bm;
    cluster.sync();
  }
  float m = s.cmax[0];
  for (int c = 1; c < C; ++c) m = fmaxf(m, s.cmax[c]);
  if (!(m > -INFINITY)) {  // nothing to draw from
    if (rank == 0 && tid == 0) a.out[row] = 0;
    return;  // the same for the whole cluster
  }
  if (k == 1 || m == INFINITY) {  // the first token alone (of infinite ones, all of score inf, the lowest index)
    int at = kNone;
    if (tmax == m)
      r.each([&](const float(&l)[kBatch], const int(&id)[kBatch]) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
          if (l[e] == m) at = min(at, id[e]);
      });
    at = warp_reduce(at, imin_op);
    if (lane == 0) s.warg[warp] = at;
    __syncthreads();
    if (warp == 0) {
      at = warp_reduce(lane < NW ? s.warg[lane] : kNone, imin_op);
      if (lane == 0) first.carg[rank] = at;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < C; ++c) at = min(at, s.carg[c]);
      a.out[row] = at;
    }
    return;
  }
  // w >= min_p as a bound on the logit: the smallest float at or above max + log(min_p)
  const float floor_l = min_p > 0.0 ? __double2float_ru((double)m + log(min_p)) : -FLT_MAX;

  auto cut_of = [&](u64 total) { return (u64)ceil(top_p * (double)total); };  // kept while the mass before is below
  // Prefix over the row's bins in s.sum (masses, or counts): the bin where the target falls, before < target <= before +
  // its own; s.bin = -1 where the row ends first. target 0: top-p's share of the total. Returns the target.
  auto find = [&](bool by_mass, u64 target) {
    constexpr int PER = kBins / NT;
    u64 w[PER], ws = 0;
    float est[PER], es = 0.f;  // tokens of the linear bins: mass over the bin's weight
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      w[i] = s.sum[tid * PER + i];
      est[i] = by_mass ? (float)w[i] * ss::ex2((tid * PER + i) * (ss::kLog2e / 64.f) - 40.f) : (float)w[i];
      ws += w[i], es += est[i];
    }
    const u64 pw = warp_scan(ws, lane);
    const float pe = warp_scan(es, lane);
    if (lane == 31) s.wsum[warp] = pw, s.west[warp] = pe;
    if (tid == 0) s.bin = -1;
    __syncthreads();
    const u64 aw = warp_scan(lane < NW ? s.wsum[lane] : 0, lane);
    const float ae = warp_scan(lane < NW ? s.west[lane] : 0.f, lane);
    if (!target) target = cut_of(__shfl_sync(0xffffffffu, aw, 31));
    u64 bw = pw - ws + __shfl_sync(0xffffffffu, aw, warp) - s.wsum[warp];
    float be = pe - es + __shfl_sync(0xffffffffu, ae, warp) - s.west[warp];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (bw < target && target <= bw + w[i]) s.bin = tid * PER + i, s.before = bw, s.est_before = be, s.est_in = est[i];
      bw += w[i], be += est[i];
    }
    __syncthreads();
    return target;
  };
  // The CTAs' histograms added: each adds a share of the bins and hands it to all.
  auto share = [&](bool by_mass) {
    cluster.sync();
    const int per = kBins / C;
    for (int i = tid; i < per; i += NT) {
      const int bin = rank * per + i;
      unsigned l[8], h[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        l[q] = h[q] = 0;
        if (q < C) {
          const Smem& o = *cluster.map_shared_rank(&s, q);
          l[q] = o.lo[bin];
          if (by_mass) h[q] = o.hi[bin];
        }
      }
      u64 w = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) w += ((u64)h[q] << 32) + l[q];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < C) cluster.map_shared_rank(&s, q)->sum[bin] = w;
    }
    cluster.sync();
  };
  auto clear = [&] {
    for (int i = tid; i < kBins; i += NT) s.lo[i] = s.hi[i] = 0;
    __syncthreads();
  };
  // A token into this CTA's list; after the pushes, all lists into the first CTA's: how many tokens there are (more than
  // kCap: the list is of no use). Ready for the next pushes.
  auto push = [&](u64 c) {
    const unsigned at = atomicAdd(&s.n_mine, 1u);
    if (at < kCap) s.mine[at] = c;
  };
  auto collected = [&] {
    __syncthreads();
    const unsigned own = s.n_mine;
    if (tid == 0) s.base = atomicAdd(&first.n, own);
    __syncthreads();
    for (unsigned i = tid; i < own && s.base + i < kCap; i += NT) first.list[s.base + i] = s.mine[i];
    if (tid == 0) s.n_mine = 0;
    cluster.sync();
    const unsigned n = first.n;
    cluster.sync();
    if (rank == 0 && tid == 0) s.n = 0;  // cluster barriers come before the next use
    return (int)min(n, (unsigned)kNone);
  };
  // The first CTA's list in descending order: bitonic, an entry a thread in registers (neighbours up to 16 away by shuffles)
  // or, beyond NT entries, in shared memory, where steps of up to 32 stay inside a warp's 64 entries.
  auto sort = [&](int n) {
    int size = 32;
    while (size < n) size <<= 1;
    if (size <= NT) {
      u64 v = tid < n ? s.list[tid] : 0;
      for (int w = 2; w <= size; w <<= 1)
        for (int d = w >> 1; d > 0; d >>= 1) {
          u64 o;
          if (d < 32) {
            o = __shfl_xor_sync(0xffffffffu, v, d);
          } else {
            __syncthreads();
            s.list[tid] = v;
            __syncthreads();
            o = s.list[tid ^ d];
          }
          const bool larger = ((tid & d) == 0) == ((tid & w) == 0);
          v = (v > o) == larger ? v : o;
        }
      __syncthreads();
      s.list[tid] = v;
      __syncthreads();
      return;
    }
    for (int i = n + tid; i < size; i += NT) s.list[i] = 0;
    __syncthreads();
    for (int w = 2; w <= size; w <<= 1)
      for (int d = w >> 1; d > 0; d >>= 1) {
        for (int i = tid; i < size / 2; i += NT) {
          const int x = (i & ~(d - 1)) * 2 + (i & (d - 1)), y = x + d;
          const u64 p = s.list[x], q = s.list[y];
          if ((p < q) == ((x & w) == 0)) s.list[x] = q, s.list[y] = p;
        }
        if (d > 32 || (d == 1 && w > 32)) __syncthreads();
        else __syncwarp();
      }
    __syncthreads();
  };
  // Mass before each of the list's first n entries and its own (LP consecutive entries a thread); the sum.
  constexpr int LP = kCap / NT;
  auto list_prefix = [&](int n, u64 (&before)[LP], u64 (&own)[LP]) {
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < LP; ++i) {
      const int at = tid * LP + i;
      own[i] = at < n ? mass(logit_of(s.list[at]), m) : 0;
      sum += own[i];
    }
    const u64 inc = warp_scan(sum, lane);
    if (lane == 31) s.wsum[warp] = inc;
    __syncthreads();
    const u64 all = warp_scan(lane < NW ? s.wsum[lane] : 0, lane);
    u64 b = inc - sum + __shfl_sync(0xffffffffu, all, warp) - s.wsum[warp];
#pragma unroll
    for (int i = 0; i < LP; ++i) before[i] = b, b += own[i];
    return __shfl_sync(0xffffffffu, all, 31);
  };
  // The CTA's best token: fp32 scores, the ones within its error of the best again in fp64.
  auto block_best = [&](const Best& b, double& score, int& index) {
    const float top = block_max(b.score);
    const bool near = b.i != kNone && (b.score == top || b.score >= top - 2.f * margin(top));
    auto join = [&](double& x, int& at) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double y = __shfl_xor_sync(0xffffffffu, x, o);
        const int i = __shfl_xor_sync(0xffffffffu, at, o);
        if (y > x || (y == x && i < at)) x = y, at = i;
      }
    };
    double x = near ? score64(b.l, b.u, temperature) : -INFINITY;
    int at = near ? b.i : kNone;
    join(x, at);
    if (lane == 0) s.wscore[warp] = x, s.warg[warp] = at;
    __syncthreads();
    score = lane < NW ? s.wscore[lane] : -INFINITY, index = lane < NW ? s.warg[lane] : kNone;
    join(score, index);
  };
  // The first CTA's list holds every token down to the last kept one: its filters, its draw. cut: top-p's, 0 for its share
  // of the list's own mass (after top-k).
  auto finish = [&](int n, u64 cut) {
    sort(n);
    if (need_k && k < n) n = (int)k;
    u64 before[LP], own[LP];
    const u64 sum = list_prefix(n, before, own);
    if (!cut) cut = need_p ? cut_of(sum) : ~0ull;
    Best b;
#pragma unroll
    for (int i = 0; i < LP; ++i) {
      const int at = tid * LP + i;
      if (at >= n || !(at == 0 || before[i] < cut)) continue;
      const u64 c = s.list[at];
      const float l = logit_of(c);
      if (l >= floor_l) {
        const float u = noise[index_of(c)];
        b.offer(score32(l, u, inv_t), l, u, index_of(c), temperature);
      }
    }
    double score;
    int index;
    block_best(b, score, index);
    if (tid == 0) a.out[row] = index;
  };

  // ---- top-k through the thread maxima
  if (need_k && k <= kFastK && k <= NT) {
    clear();
    if (tmax > -INFINITY) atomicAdd(&s.lo[linear_bin(tmax, m)], 1u);
    __syncthreads();
    for (int i = tid; i < kBins; i += NT) s.sum[i] = s.lo[i];
    __syncthreads();
    find(false, (u64)k);
    if (tid < C) cluster.map_shared_rank(&s, tid)->cbin[rank] = s.bin < 0 ? kBins : s.bin;
    cluster.sync();
    int bound = s.cbin[0];  // k thread maxima of one CTA lie in bins up to its bound
    for (int c = 1; c < C; ++c) bound = min(bound, s.cbin[c]);
    // bins up to `bound` lie within (bound + 1) / 64 of the maximum; the last bin has no lower end
    const float reach = bound >= kBins - 1 ? INFINITY : (bound + 1) * (1.f / 64.f);
    r.each([&](const float(&l)[kBatch], const int(&id)[kBatch]) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) any |= m - l[e] <= reach;
      if (!any) return;
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (m - l[e] <= reach && l[e] > -INFINITY) push(composite(clean(l[e]), id[e]));
    });
    const int n = collected();
    if (n <= kCap) {
      if (rank == 0) finish(n, 0);
      return;
    }
  }

  u64 keep = 0;  // tokens with a composite below are cut
  // ---- one cut: the last token with fewer than k tokens (less than top-p's share of the mass) before it, among those
  // from `keep` on; true where that finished the row.
  auto descend = [&](bool by_mass) {
    u64 target = by_mass ? 0 : (u64)k, before = 0, prefix = 0;
    // the group of tokens that is being cut: linear bin `lin` (-1: all), composite >> shift == prefix
    int lin = -1, shift = 64;
    for (;;) {
      const int low = shift > 11 ? shift - 11 : 0, last = (1 << (shift - low)) - 1;
      auto bin_of = [&](int i, float l) {  // -1: outside the group
        const int b = linear_bin(l, m);
        if (!(l > -INFINITY)) return -1;
        if (lin < 0) return keep && composite(clean(l), i) < keep ? -1 : b;
        if (b != lin) return -1;
        const u64 c = composite(clean(l), i);
        if (c < keep || (shift < 64 && (c >> shift) != prefix)) return -1;
        return last - ((int)(c >> low) & last);
      };
      clear();
      // adds a batch to the histogram, b < 0 left out: all first words, then the carries
      auto add = [&](const int(&b)[kBatch], const uint2(&w)[kBatch]) {
        unsigned old[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) old[e] = b[e] >= 0 ? atomicAdd(&s.lo[b[e]], w[e].x) : 0;
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const unsigned wh = w[e].y + (old[e] + w[e].x < old[e]);
          if (b[e] >= 0 && wh) atomicAdd(&s.hi[b[e]], wh);
        }
      };
      if (lin < 0 && !keep && by_mass) {  // the usual case without what the others ask
        r.each([&](const float(&l)[kBatch], const int(&)[kBatch]) {
          int b[kBatch];
          uint2 w[kBatch];
#pragma unroll
          for (int e = 0; e < kBatch; ++e) {
            b[e] = l[e] > -INFINITY ? linear_bin(l[e], m) : -1;
            w[e] = mass2(l[e], m);
          }
          add(b, w);
        });
      } else {
        r.each([&](const float(&l)[kBatch], const int(&id)[kBatch]) {
          int b[kBatch];
          uint2 w[kBatch];
#pragma unroll
          for (int e = 0; e < kBatch; ++e) {
            b[e] = bin_of(id[e], l[e]);
            w[e] = by_mass ? mass2(l[e], m) : make_uint2(1, 0);
          }
          add(b, w);
        });
      }
      share(by_mass);
      target = find(by_mass, lin < 0 && by_mass ? 0 : target - before) + before;
      const int bin = s.bin;
      if (bin < 0) return false;  // every token is kept
      const u64 in_bin = target - before - s.before;  // the target within the bin
      const float est_before = s.est_before, est_in = s.est_in;
      // the whole list down to the bin, where it should fit
      if (lin < 0 && est_before + est_in < 0.9f * kCap) {
        r.each([&](const float(&l)[kBatch], const int(&id)[kBatch]) {
#pragma unroll
          for (int e = 0; e < kBatch; ++e)
            if ((unsigned)bin_of(id[e], l[e]) <= (unsigned)bin) push(composite(clean(l[e]), id[e]));
        });
        const int n = collected();
        if (n <= kCap) {
          if (rank == 0) finish(n, by_mass ? target : 0);
          return true;
        }
      }
      // the bin alone (an estimate of a digit's bin is its linear bin's: it is collected when that fits, or is tried)
      if (lin >= 0 || est_in < 1.1f * kCap) {
        cluster.sync();
        r.each([&](const float(&l)[kBatch], const int(&id)[kBatch]) {
          unsigned in = 0;
          if (lin < 0) {
#pragma unroll
            for (int e = 0; e < kBatch; ++e) in |= (unsigned)(linear_bin(l[e], m) == bin) << e;
          } else {
#pragma unroll
            for (int e = 0; e < kBatch; ++e) in |= (unsigned)(linear_bin(l[e], m) == lin) << e;
          }
          if (!in) return;
#pragma unroll
          for (int e = 0; e < kBatch; ++e)
            if ((in >> e & 1) && bin_of(id[e], l[e]) == bin) push(composite(clean(l[e]), id[e]));
        });
        const int n = collected();
        if (n <= kCap) {
          if (rank == 0) {
            sort(n);
            if (by_mass) {
              u64 b[LP], own[LP];
              list_prefix(n, b, own);
#pragma unroll
              for (int j = 0; j < LP; ++j) {
                const int at = tid * LP + j;
                if (at < n && b[j] < in_bin && (at == n - 1 || b[j] + own[j] >= in_bin)) s.cut = s.list[at];
              }
            } else if (tid == 0) {
              s.cut = s.list[in_bin - 1];
            }
            __syncthreads();
            const u64 cut = s.cut;
            if (tid < C) cluster.map_shared_rank(&s, tid)->cut = cut;
          }
          cluster.sync();
          keep = s.cut;
          return false;
        }
      }
      before += s.before;
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
  const unsigned keep_key = (unsigned)(keep >> 32);
  const float keep_l = keep ? fmaxf(unordered(keep_key), floor_l) : floor_l;
  float top = -INFINITY;  // of the warp: a lane's own best alone lets some lane of 32 through nearly every time
  r.each([&](const float(&l)[kBatch], const int(&id)[kBatch]) {
    float u[kBatch], sc[kBatch], most = l[0];
#pragma unroll
    for (int e = 1; e < kBatch; ++e) most = fmaxf(most, l[e]);
    if (!(most >= keep_l)) return;
    unsigned in = 0;
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const bool on = l[e] >= keep_l && (l[e] > keep_l || composite(clean(l[e]), id[e]) >= keep);
      in |= (unsigned)on << e;
      u[e] = on ? noise[id[e]] : 0.f;
    }
    const float bar = top - margin(top);
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      sc[e] = score32(l[e], u[e], inv_t);
      if (sc[e] < bar) in &= ~(1u << e);  // out of reach (what is beyond fp32 is not)
    }
    if (in) {
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (in >> e & 1) b.offer(sc[e], l[e], u[e], id[e], temperature);
    }
    const unsigned here = __activemask();
    if (__ballot_sync(here, in != 0)) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float y = __shfl_xor_sync(here, b.score, o);
        if (here >> (lane ^ o) & 1) top = fmaxf(top, y);
      }
      top = fmaxf(top, b.score);
    }
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
