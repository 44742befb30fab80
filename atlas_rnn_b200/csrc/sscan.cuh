// Selective state space scan: per batch row, channel d and state n
//   dt_t = softplus(delta_t + bias) (or delta_t + bias),  a_t = exp(dt_t A[d,n]),
//   h_t  = a_t h_{t-1} + dt_t u_t B_t[n],  y_t = sum_n C_t[n] h_t + D u_t,  out_t = y_t silu(z_t),
// and its backward. The scalar-gated scans of scan_op.cuh share one gate over the whole state; here
// every (channel, state) pair has its own, so the exponentials, one per (token, channel, state), set
// the floor: 16 per cycle and SM on the special-function unit, against about 20 bytes of traffic
// per (token, channel). At B 4, T 8192, D 1536, N 16, bf16 (358 us of exponentials, one a state and direction): forward
// 255 us for the chunks' ends and 350 for the outputs, backward 257 and 986. The ends passes keep the special-function unit
// 80% busy; the forward's main pass 65% with an issue slot used every other cycle; the backward's 43%, with 12 warps an SM
// for its registers and two exponentials a state (a_t is computed again).
//
// Layout of the work: a channel's states lie across LPC = NP / kSpt lanes (NP: the state count padded to a power of two
// with A = B = C = 0 columns, whose states stay 0), and a lane holds the states of MC neighbouring channels: a load from
// shared memory returns 4 bytes a lane and cycle, so B and C serve the lane's MC channels, dt and dt u its kSpt states
// (one channel a lane cost 3.5 load cycles of the SM a state-update of a warp, above the exponential's 2). A
// warp walks the time axis in tiles of kTT steps. Everything is the warp's own, so a tile costs no block barrier: rows
// arrive by cp.async one tile ahead and become dt, dt u, B, C in fp32; arithmetic is packed fp32 pairs over
// neighbouring states; the sums over a channel's lanes are transposed reductions (LPC values over LPC lanes in
// LPC - 1 exchanges). Lengths: a step at or past its row's length is not read and writes 0. States, sums and
// gates are fp32; what is written in the rows' type is rounded once, from fp32.
//
// When the rows and channels do not fill the machine, the time axis is cut into chunks: a first
// pass leaves each chunk's own end state (from zero) and its sum of dt, k_sscan_carry turns them into the states
// that enter the chunks (each earlier one decayed by exp(A sum dt)), and the pass over the outputs starts from those.
// That pays the exponentials twice.
#pragma once
#include <cfloat>
#include <type_traits>

#include "row_ops.cuh"

namespace atlas {
namespace ss {

// Channels per lane, forward and backward. Forward 4: fewer shared-memory loads and instructions a state (measured at
// B 4, T 8192, D 1536, N 16, bf16: 350 us; 2 with as many or more warps 5-15% more). Backward 2: the states of
// kTT steps stay in 168 registers (986 us; 4 needs 255 registers: 4-15% more), but for spills of 8-144 bytes (N over 32:
// 640-896). Wide states take 4: 2 would leave a warp less than 16 bytes of a row.
constexpr int kMcFwd = 4;
template <int NP>
constexpr int kMcBwd = NP < 64 ? 2 : 4;
constexpr int kTT = 8;     // steps per tile; training keeps the state before each
constexpr int kSpt = 4;    // states per lane
constexpr int kWarps = 4;   // per CTA
constexpr int kFwdCtas = 4, kBwdCtas = 3;  // resident on an SM (registers: 128 and 168 a thread)

struct ScanArgs {
  const void *u, *delta, *z, *Bm, *Cm, *dout;
  int64_t u_sb, u_st, d_sb, d_st, z_sb, z_st, o_sb, o_st;  // element strides (batch, step); channels are dense
  int64_t B_sb, B_st, B_sg, C_sb, C_st, C_sg;              // (batch, step, group); states are dense
  const float *A, *D, *bias, *h0;
  const int* len;
  void* out;       // [B, T, Dm]
  float* hT;       // [B, Dm, N]
  float* hsave;    // [B, ceil(T / kTT), Dm, NP]
  float* part_h;   // [B, nchunk, Dm, NP]  chunk end states (backward: start adjoints)
  float* part_dt;  // [B, nchunk, Dm]      chunk sums of dt
  // backward
  const float* dhT;  // [B, Dm, N] or null
  void *du, *ddelta, *dz;  // [B, T, Dm]
  float* dbc;        // [tiles, B, T, 2, NP] per channel tile: d B, d C (null: not wanted)
  float* part_dA;    // [B * nchunk, Dm, NP]
  float* part_dD;    // [B * nchunk, 2, Dm]  d D, d bias
  float* dh0;        // [B, Dm, N] or null
  int64_t T;
  int Bsz, Dm, N, G, softplus, chunk, nchunk;  // chunk: steps per chunk, a multiple of kTT
  int vec;   // every row tensor allows whole-vector accesses (16 bytes or the thread's share)
  int vecbc; // B and C allow 16-byte (backward: 4-element) accesses
  int pair;  // the output's rows allow two-element accesses at even channels
};

// ---- shared by the passes -------------------------------------------------
template <int NP, int MC>
struct Shape {
  static constexpr int LPC = NP / kSpt;      // lanes across a channel's states
  static constexpr int Q = 32 / LPC;         // channel groups in a warp
  static constexpr int CH = Q * MC;          // channels of a warp
  static constexpr int PC = CH / 2 < 32 ? CH / 2 : 32;  // row phases: a lane takes two channels of a row ..
  static constexpr int PR = 32 / PC;         // .. PR rows at a time
  static constexpr int SY = LPC > MC ? LPC / MC : 1;    // steps per reduction over a channel's lanes
  static constexpr int SB = Q > kSpt ? Q / kSpt : 1;    // steps per reduction over the warp's channel groups
  static_assert(PC * 2 == CH && kTT % PR == 0 && SY <= kTT && SB <= kTT, "tile");
};

// A warp's place in the problem.
template <int CH>
struct Place {
  int b, g, nc, tile;  // nc: channels it really has; tile: the CTA's channel tile index over all groups
  int64_t d0, len;
  __device__ Place(const ScanArgs& a, int warp) {
    const int Dg = a.Dm / a.G, tiles = (Dg + CH * kWarps - 1) / (CH * kWarps);
    b = blockIdx.x / (tiles * a.G);
    tile = blockIdx.x - b * tiles * a.G;
    g = tile / tiles;
    const int c = ((tile - g * tiles) * kWarps + warp) * CH;
    nc = Dg - c < CH ? (Dg - c < 0 ? 0 : Dg - c) : CH;
    d0 = (int64_t)g * Dg + (nc ? c : 0);
    len = row_len(a.len, b, a.T);
  }
};

// A lane's MC x kSpt block of per-(channel, state) values, as pairs over neighbouring states.
template <int MC>
struct Block {
  f2 v[MC][kSpt / 2];
  // value(c, i) of the lane's channel c and state i
  template <class F>
  __device__ __forceinline__ void fill(F value) {
#pragma unroll
    for (int c = 0; c < MC; ++c)
#pragma unroll
      for (int p = 0; p < kSpt / 2; ++p) v[c][p] = pk(value(c, 2 * p), value(c, 2 * p + 1));
  }
  __device__ __forceinline__ float at(int c, int i) const {
    const float2 x = up(v[c][i / 2]);
    return i % 2 ? x.y : x.x;
  }
};

// A in units of log2. -inf is the lowest finite value: dt A is 0, not NaN, at the steps that a tile or a chunk has too
// many, whose dt is 0.
__device__ __forceinline__ float log2_decay(float A) {
  const float v = A * kLog2e;
  return v < -FLT_MAX ? -FLT_MAX : v;
}
// A [Dm, N] in units of log2.
template <int MC, int CH>
__device__ __forceinline__ void load_A(const ScanArgs& a, const Place<CH>& w, int c4, int n4, Block<MC>& A) {
  A.fill([&](int c, int i) {
    return c4 + c < w.nc && n4 + i < a.N ? log2_decay(a.A[(w.d0 + c4 + c) * a.N + n4 + i]) : 0.f;
  });
}
// A state [B, Dm, N] (null: zeros).
template <int MC, int CH>
__device__ __forceinline__ void load_state(const ScanArgs& a, const Place<CH>& w, const float* s, int c4, int n4,
                                           Block<MC>& h) {
  h.fill([&](int c, int i) {
    return s && c4 + c < w.nc && n4 + i < a.N ? s[((int64_t)w.b * a.Dm + w.d0 + c4 + c) * a.N + n4 + i] : 0.f;
  });
}
template <int MC, int CH>
__device__ __forceinline__ void store_state(const ScanArgs& a, const Place<CH>& w, float* s, int c4, int n4,
                                            const Block<MC>& h) {
#pragma unroll
  for (int c = 0; c < MC; ++c)
#pragma unroll
    for (int i = 0; i < kSpt; ++i)
      if (c4 + c < w.nc && n4 + i < a.N) s[((int64_t)w.b * a.Dm + w.d0 + c4 + c) * a.N + n4 + i] = h.at(c, i);
}
// Channel rows of NP padded states (16-byte pieces).
template <int NP, int MC>
__device__ __forceinline__ void store_rows(float* rows, int nc, int c4, int n4, const Block<MC>& h) {
#pragma unroll
  for (int c = 0; c < MC; ++c)
    if (c4 + c < nc)
      *reinterpret_cast<ulonglong2*>(rows + (int64_t)(c4 + c) * NP + n4) = make_ulonglong2(h.v[c][0], h.v[c][1]);
}
template <int NP, int MC>
__device__ __forceinline__ void load_rows(const float* rows, int nc, int c4, int n4, Block<MC>& h) {
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    ulonglong2 x = make_ulonglong2(0, 0);
    if (c4 + c < nc) x = *reinterpret_cast<const ulonglong2*>(rows + (int64_t)(c4 + c) * NP + n4);
    h.v[c][0] = x.x, h.v[c][1] = x.y;
  }
}
// A lane's channels in a row of fp32, each as a pair.
template <int MC>
struct Chans {
  f2 v[MC];
  __device__ __forceinline__ explicit Chans(const float* p) {
    if constexpr (MC == 4) {
      const float4 x = *reinterpret_cast<const float4*>(p);
      v[0] = both(x.x), v[1] = both(x.y), v[2] = both(x.z), v[3] = both(x.w);
    } else {
      const float2 x = *reinterpret_cast<const float2*>(p);
      v[0] = both(x.x), v[1] = both(x.y);
    }
  }
};
// A [kTT, NP] tile in fp32.
template <class IO, int NP>
__device__ __forceinline__ void widen(float (*dst)[NP], const IO* raw, int lane) {
#pragma unroll
  for (int k = 0; k < kTT * NP; k += 64) st2(&dst[0][0] + k + lane * 2, ld2(raw + k + lane * 2));
}
// A lane's four states in a row of fp32.
struct States {
  f2 v[kSpt / 2];
  __device__ __forceinline__ explicit States(const float* p) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(p);
    v[0] = x.x, v[1] = x.y;
  }
};
// One step of the recurrence.
template <int MC>
__device__ __forceinline__ void advance(Block<MC>& h, const Block<MC>& from, const Block<MC>& A, const Chans<MC>& dt,
                                        const Chans<MC>& du, const States& B) {
#pragma unroll
  for (int c = 0; c < MC; ++c)
#pragma unroll
    for (int p = 0; p < kSpt / 2; ++p)
      h.v[c][p] = fma2(ex2_2(mul2(A.v[c][p], dt.v[c])), from.v[c][p], mul2(du.v[c], B.v[p]));
}
// The lane's share of sum_n C h, per channel.
template <int MC>
__device__ __forceinline__ void dot(float* y, const Block<MC>& h, const States& C) {
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const float2 v = up(fma2(C.v[1], h.v[c][1], mul2(C.v[0], h.v[c][0])));
    y[c] = v.x + v.y;
  }
}
// Two neighbouring elements of a row written: both where the warp's tile is whole and pairs are aligned.
template <class IO>
__device__ __forceinline__ void store2(IO* o, f2 v, bool whole, bool c0, bool c1) {
  if (whole) {
    st2(o, v);
  } else {
    const float2 x = up(v);
    if (c0) from_f(o[0], x.x);
    if (c1) from_f(o[1], x.y);
  }
}
// Sum over the lanes that share the column pair of a row phase.
template <int PC>
__device__ __forceinline__ f2 over_rows(f2 x) {
#pragma unroll
  for (int o = PC; o < 32; o <<= 1) x = add2(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// ---- forward --------------------------------------------------------------
template <class IO, int NP, bool ENDS, bool Z>
struct FwdSmem {  // one warp's
  static constexpr int kRows = Z ? 3 : 2, kBC = ENDS ? 1 : 2, CH = Shape<NP, kMcFwd>::CH;
  struct Raw {  // a tile as it lies in memory
    alignas(16) IO rows[kRows][kTT][CH];  // delta, u, z
    alignas(16) IO bc[kBC][kTT][NP];
  };
  Raw raw[2];
  alignas(16) float dt[kTT][CH];
  alignas(16) float du[kTT][CH];
  alignas(16) float b[kTT][NP];
  alignas(16) float c[ENDS ? 1 : kTT][NP];
  alignas(16) float y[ENDS ? 1 : kTT][CH];
};

// grid (batch x groups x channel tiles, chunks). ENDS: only the chunk's end state and sum of dt.
template <class IO, int NP, bool ENDS, bool Z>
__global__ void __launch_bounds__(32 * kWarps, kFwdCtas) k_sscan_fwd(const ScanArgs a) {
  using SM = FwdSmem<IO, NP, ENDS, Z>;
  constexpr int MC = kMcFwd;
  using S = Shape<NP, MC>;
  constexpr int LPC = S::LPC, CH = S::CH, PC = S::PC, PR = S::PR, SY = S::SY;
  extern __shared__ __align__(16) unsigned char sm_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPC;
  SM& sm = reinterpret_cast<SM*>(sm_raw)[warp];
  const Place<CH> w(a, warp);
  if (!w.nc) return;  // warps do not wait for one another here
  const int chunk = blockIdx.y, c4 = lane / LPC * MC, n4 = l * kSpt;
  const int64_t t_lo = (int64_t)chunk * a.chunk, t_hi = t_lo + a.chunk < a.T ? t_lo + a.chunk : a.T;
  const int64_t t_live = t_hi < w.len ? t_hi : w.len;
  const int pc = lane % PC * 2, pr = lane / PC;
  using Rows = Feed<IO, kTT, CH>;
  using Cols = Feed<IO, kTT, NP>;
  Rows fd((const IO*)a.delta + w.b * a.d_sb + t_lo * a.d_st + w.d0, a.d_st, w.nc, a.vec, lane);
  Rows fu((const IO*)a.u + w.b * a.u_sb + t_lo * a.u_st + w.d0, a.u_st, w.nc, a.vec, lane);
  Rows fz(Z ? (const IO*)a.z + w.b * a.z_sb + t_lo * a.z_st + w.d0 : nullptr, a.z_st, w.nc, a.vec, lane);
  Cols fb((const IO*)a.Bm + w.b * a.B_sb + w.g * a.B_sg + t_lo * a.B_st, a.B_st, a.N, a.vecbc, lane);
  Cols fc((const IO*)a.Cm + w.b * a.C_sb + w.g * a.C_sg + t_lo * a.C_st, a.C_st, a.N, a.vecbc, lane);
  auto fetch = [&](int rows, int s) {  // the next tile
    auto& r = sm.raw[s];
    if (a.vec) {
      fd.vectors(&r.rows[0][0][0], a.d_st, rows, lane);
      fu.vectors(&r.rows[1][0][0], a.u_st, rows, lane);
      if (Z) fz.vectors(&r.rows[SM::kRows - 1][0][0], a.z_st, rows, lane);
    } else {
      fd.elements(&r.rows[0][0][0], a.d_st, rows, lane);
      fu.elements(&r.rows[1][0][0], a.u_st, rows, lane);
      if (Z) fz.elements(&r.rows[SM::kRows - 1][0][0], a.z_st, rows, lane);
    }
    if (a.vecbc) {
      fb.vectors(&r.bc[0][0][0], a.B_st, rows, lane);
      if (!ENDS) fc.vectors(&r.bc[SM::kBC - 1][0][0], a.C_st, rows, lane);
    } else {
      fb.elements(&r.bc[0][0][0], a.B_st, rows, lane);
      if (!ENDS) fc.elements(&r.bc[SM::kBC - 1][0][0], a.C_st, rows, lane);
    }
    fd.p += kTT * a.d_st, fu.p += kTT * a.u_st, fb.p += kTT * a.B_st;
    if (Z) fz.p += kTT * a.z_st;
    if (!ENDS) fc.p += kTT * a.C_st;
    cp_commit();
  };
  int left = t_live > t_lo ? (int)(t_live - t_lo) : 0;  // steps to walk
  if (left) fetch(left, 0);

  Block<MC> A, h;
  load_A(a, w, c4, n4, A);
  if (!ENDS && a.nchunk > 1)
    load_rows<NP>(a.part_h + (((int64_t)w.b * a.nchunk + chunk) * a.Dm + w.d0) * NP, w.nc, c4, n4, h);
  else
    load_state(a, w, ENDS ? nullptr : a.h0, c4, n4, h);
  const bool c0 = pc < w.nc, c1 = pc + 1 < w.nc, whole = a.pair && w.nc == CH;
  IO* out = (IO*)a.out + (w.b * a.T + t_lo + pr) * a.Dm + w.d0 + pc;
  const f2 bias = pk(c0 && a.bias ? a.bias[w.d0 + pc] : 0.f, c1 && a.bias ? a.bias[w.d0 + pc + 1] : 0.f);
  const f2 skip = pk(c0 && a.D ? a.D[w.d0 + pc] : 0.f, c1 && a.D ? a.D[w.d0 + pc + 1] : 0.f);
  f2 sdt = 0;
  const int64_t nblk = (a.T + kTT - 1) / kTT;
  float* hs = a.hsave ? a.hsave + ((w.b * nblk + t_lo / kTT) * a.Dm + w.d0) * NP : nullptr;

  for (int s = 0; left > 0; left -= kTT, s ^= 1) {
    const int rows = left;  // of this tile, where below kTT
    if (left > kTT) {
      fetch(left - kTT, s ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncwarp();
    auto& raw = sm.raw[s];
#pragma unroll
    for (int k = 0; k < kTT; k += PR) {
      const int tt = pr + k;
      f2 x = add2(ld2(&raw.rows[0][tt][pc]), bias);
      if (a.softplus) x = softplus_2(x);
      if (tt >= rows) x = 0;
      if (ENDS) sdt = add2(sdt, x);
      st2(&sm.dt[tt][pc], x);
      st2(&sm.du[tt][pc], mul2(x, ld2(&raw.rows[1][tt][pc])));
    }
    widen<IO, NP>(sm.b, &raw.bc[0][0][0], lane);
    if (!ENDS) widen<IO, NP>(sm.c, &raw.bc[SM::kBC - 1][0][0], lane);
    __syncwarp();
    if (!ENDS && hs) {
      store_rows<NP>(hs, w.nc, c4, n4, h);
      hs += (int64_t)a.Dm * NP;
    }

#pragma unroll
    for (int ts = 0; ts < kTT; ts += SY) {
      float p[SY * MC];
#pragma unroll
      for (int j = 0; j < SY; ++j) {
        const int tt = ts + j;
        advance(h, h, A, Chans<MC>(&sm.dt[tt][c4]), Chans<MC>(&sm.du[tt][c4]), States(&sm.b[tt][n4]));
        if (!ENDS) dot(p + j * MC, h, States(&sm.c[tt][n4]));
      }
      if (!ENDS) {
        reduce_part<SY * MC, LPC, 1>(p, lane);
        constexpr int R = SY * MC / LPC;  // values a lane keeps: its channels l R .. of step ts + l R / MC
#pragma unroll
        for (int r = 0; r < R; ++r) sm.y[ts + l * R / MC][c4 + l * R % MC + r] = p[r];
      }
    }
    __syncwarp();
    if (!ENDS) {
      auto rows_out = [&](auto whole_tile_) {  // every row and channel pair of the tile, or those that there are
        constexpr bool whole_tile = decltype(whole_tile_)::value;
#pragma unroll
        for (int k = 0; k < kTT; k += PR) {
          const int tt = pr + k;
          f2 y = fma2(skip, ld2(&raw.rows[1][tt][pc]), ld2(&sm.y[tt][pc]));
          if (Z) {
            const f2 z = ld2(&raw.rows[SM::kRows - 1][tt][pc]);
            y = mul2(y, mul2(z, sigmoid_2(z)));
          }
          if (whole_tile) st2(out + k * (int64_t)a.Dm, y);
          else if (tt < rows) store2(out + k * (int64_t)a.Dm, y, whole, c0, c1);
        }
      };
      if (whole && rows >= kTT) rows_out(std::true_type());
      else rows_out(std::false_type());
      out += kTT * (int64_t)a.Dm;
      __syncwarp();  // the fetch after next writes these rows
    }
  }
  if (ENDS) {
    const int64_t at = ((int64_t)w.b * a.nchunk + chunk) * a.Dm + w.d0;
    store_rows<NP>(a.part_h + at * NP, w.nc, c4, n4, h);
    const float2 v = up(over_rows<PC>(sdt));
    if (pr == 0 && c0) a.part_dt[at + pc] = v.x;
    if (pr == 0 && c1) a.part_dt[at + pc + 1] = v.y;
  } else {
    out = (IO*)a.out + w.b * a.T * a.Dm + w.d0 + pc;
    for (int64_t t = (t_live > t_lo ? t_live : t_lo) + pr; t < t_hi; t += PR)  // zeros past the length
      store2(out + t * a.Dm, 0, whole, c0, c1);
    if (chunk == a.nchunk - 1) store_state(a, w, a.hT, c4, n4, h);
  }
}

// The chunks' records in order (BACK: from the last): record c, the end state from zero, becomes the state that enters
// chunk c. A thread takes 4 states of a channel, its loads kAhead records ahead of the serial chain: as a prologue of
// every chunk's warps it cost 42 us of 70 at 64 chunks.
constexpr int kCarryThr = 128, kAhead = 8;
// 2^x h + e of a chunk that multiplies the state by 2^x. Where the states grow (dt A > 0), 2^x may overflow although its
// product with h does not: by halves, and a state of 0 stays out of it.
__device__ __forceinline__ float past_chunk(float x, float h, float e) {
  if (x < 127.f) return fmaf(ex2(x), h, e);
  const float half = ex2(0.5f * x);
  return h == 0.f ? e : fmaf(h * half, half, e);
}
template <int NP, bool BACK>
__global__ void __launch_bounds__(kCarryThr) k_sscan_carry(const ScanArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kCarryThr + threadIdx.x, row = i / (NP / 4);  // b * Dm + d
  if (row >= (int64_t)a.Bsz * a.Dm) return;
  const int n4 = (int)(i % (NP / 4)) * 4, b = (int)(row / a.Dm), d = (int)(row % a.Dm);
  const float* s = BACK ? a.dhT : a.h0;
  float A[4], h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    A[k] = n4 + k < a.N ? log2_decay(a.A[(int64_t)d * a.N + n4 + k]) : 0.f;
    h[k] = s && n4 + k < a.N ? s[row * a.N + n4 + k] : 0.f;
  }
  // the record that enters last has no end state: chunk nchunk - 1 (BACK: 0)
  const int64_t step = (BACK ? -1 : 1) * (int64_t)a.Dm, first = (int64_t)b * a.nchunk * a.Dm + d +
                                                                 (BACK ? (a.nchunk - 1) * (int64_t)a.Dm : 0);
  for (int c0 = 0; c0 < a.nchunk; c0 += kAhead) {
    float4 e[kAhead];
    float dt[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const bool on = c0 + k < a.nchunk - 1;
      const int64_t at = first + (on ? c0 + k : 0) * step;
      e[k] = *reinterpret_cast<const float4*>(a.part_h + at * NP + n4);
      dt[k] = a.part_dt[at];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (c0 + k >= a.nchunk) break;
      *reinterpret_cast<float4*>(a.part_h + (first + (c0 + k) * step) * NP + n4) = make_float4(h[0], h[1], h[2], h[3]);
      h[0] = past_chunk(A[0] * dt[k], h[0], e[k].x);
      h[1] = past_chunk(A[1] * dt[k], h[1], e[k].y);
      h[2] = past_chunk(A[2] * dt[k], h[2], e[k].z);
      h[3] = past_chunk(A[3] * dt[k], h[3], e[k].w);
    }
  }
}

// ---- one token ------------------------------------------------------------
// T = 1 without a backward: a thread takes 4 neighbouring states (one 16-byte read and write of the state, which is the
// traffic) of R batch rows, whose loads are all in flight together; LPC = NP / 4 lanes a channel. A, D and bias are read
// once for the R rows (1 or 4). What a row needs once a channel (dt, the gate, the output) is done by one of the channel's lanes, R
// rows by as many lanes. grid (channel blocks, row blocks).
constexpr int kStepThr = 128;
// V4: 16-byte accesses to A and the states, 4-element ones to B and C (N a multiple of 4)
template <class IO, int NP, int R, bool V4>
__global__ void __launch_bounds__(kStepThr) k_sscan_step(const ScanArgs a) {
  constexpr int LPC = NP / 4, L = LPC < R ? LPC : R, RPL = R / L;  // lanes that take a row's own part; rows of each
  const int l = threadIdx.x % LPC, d = blockIdx.x * (kStepThr / LPC) + threadIdx.x / LPC, n4 = l * 4;
  const bool on = d < a.Dm && (!V4 || n4 < a.N);
  const int dd = d < a.Dm ? d : 0, nn = V4 && n4 < a.N ? n4 : 0, g = a.G == 1 ? 0 : dd / (a.Dm / a.G);
  const int64_t b0 = (int64_t)blockIdx.y * R;
  const int left = a.Bsz - b0 < R ? (int)(a.Bsz - b0) : R, k0 = l % L * RPL;  // rows there are; the lane's first one
  auto four = [&](const float* p) {  // states n4 .. n4 + 3 of a row
    if (V4) return *reinterpret_cast<const float4*>(p + nn);
    return make_float4(n4 < a.N ? p[n4] : 0.f, n4 + 1 < a.N ? p[n4 + 1] : 0.f, n4 + 2 < a.N ? p[n4 + 2] : 0.f,
                       n4 + 3 < a.N ? p[n4 + 3] : 0.f);
  };
  auto cols = [&](const IO* p) {
    if (V4) return *reinterpret_cast<const Vec<IO, 4>*>(p + nn);
    return load_row<IO, 4>(p, n4, a.N, 0);
  };
  // all loads first, of rows that exist (what a dead row holds is dropped below), nothing used before the last is issued
  const float4 A = four(a.A + (int64_t)dd * a.N);
  const float bias = a.bias ? a.bias[dd] : 0.f, skip = a.D ? a.D[dd] : 0.f;
  const float* h0 = a.h0 ? a.h0 + (b0 * a.Dm + dd) * a.N : nullptr;
  const IO *pB = (const IO*)a.Bm + b0 * a.B_sb + g * a.B_sg, *pC = (const IO*)a.Cm + b0 * a.C_sb + g * a.C_sg;
  float4 h[R];
  Vec<IO, 4> B[R], C[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t k = r < left ? r : 0;
    h[r] = h0 ? four(h0 + k * a.Dm * a.N) : make_float4(0.f, 0.f, 0.f, 0.f);
    B[r] = cols(pB + k * a.B_sb);
    C[r] = cols(pC + k * a.C_sb);
  }
  IO ru[RPL], rd[RPL], rz[RPL];
  int len[RPL];
#pragma unroll
  for (int j = 0; j < RPL; ++j) {
    const int64_t b = b0 + (k0 + j < left ? k0 + j : 0);
    ru[j] = ((const IO*)a.u)[b * a.u_sb + dd];
    rd[j] = ((const IO*)a.delta)[b * a.d_sb + dd];
    rz[j] = a.z ? ((const IO*)a.z)[b * a.z_sb + dd] : ru[j];
    len[j] = a.len ? a.len[b] : 1;
  }
  float u[RPL], x[RPL], xu[RPL];
#pragma unroll
  for (int j = 0; j < RPL; ++j) {
    u[j] = to_f(ru[j]);
    x[j] = to_f(rd[j]) + bias;
    if (a.softplus) x[j] = softplus(x[j]);
    xu[j] = x[j] * u[j];
  }
  const float Av[4] = {log2_decay(A.x), log2_decay(A.y), log2_decay(A.z), log2_decay(A.w)};
  float y[R];
  float* ho = a.hT + (b0 * a.Dm + d) * a.N + n4;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float xr = __shfl_sync(0xffffffffu, x[r % RPL], r / RPL, LPC), xur = __shfl_sync(0xffffffffu, xu[r % RPL], r / RPL, LPC);
    const bool live = !a.len || __shfl_sync(0xffffffffu, len[r % RPL], r / RPL, LPC) > 0;
    float hv[4] = {h[r].x, h[r].y, h[r].z, h[r].w};
    y[r] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = fmaf(ex2(Av[i] * xr), hv[i], xur * to_f(B[r].v[i]));
      if (live) hv[i] = v;
      if (V4 ? on : n4 + i < a.N) y[r] = fmaf(to_f(C[r].v[i]), hv[i], y[r]);
    }
    if (d < a.Dm && r < left) {
      float* o = ho + (int64_t)r * a.Dm * a.N;
      if (V4) {
        if (on) *reinterpret_cast<float4*>(o) = make_float4(hv[0], hv[1], hv[2], hv[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n4 + i < a.N) o[i] = hv[i];
      }
    }
  }
  // lanes 2 apart first, then 1, then 4 and more, whatever R is: a row's result does not depend on the rows beside it
  reduce_part<R, L, 1>(y, threadIdx.x & 31);
  if (R == 1) {
#pragma unroll
    for (int o = LPC < 4 ? LPC / 2 : 2; o > 0; o >>= 1) y[0] += __shfl_xor_sync(0xffffffffu, y[0], o);
  }
#pragma unroll
  for (int o = R == 1 ? 4 : L; o < LPC; o <<= 1)
#pragma unroll
    for (int j = 0; j < RPL; ++j) y[j] += __shfl_xor_sync(0xffffffffu, y[j], o);
  if (l >= L || d >= a.Dm) return;
#pragma unroll
  for (int j = 0; j < RPL; ++j) {
    if (k0 + j >= left) continue;
    float v = fmaf(skip, u[j], y[j]);
    if (a.z) {
      const float z = to_f(rz[j]);
      v *= z * sigmoid(z);
    }
    from_f(((IO*)a.out)[(b0 + k0 + j) * a.Dm + d], len[j] > 0 ? v : 0.f);
  }
}

// ---- backward -------------------------------------------------------------
// With dy = dout silu(z) and g_t the gradient reaching h_t:
//   g_t = C_t dy_t + a_{t+1} g_{t+1} (from dhT),  q_t = a_t g_t reaches h_{t-1};
//   dC_t = sum_d dy_t h_t,  dB_t = sum_d g_t dt_t u_t,  s1_t = sum_n g_t B_t,  w = g_t a_t h_{t-1},
//   du = dt s1 + D dy,  d dt = sum_n w A + u s1,  dA = sum_t w dt,  ddelta = d dt sigmoid(delta + bias),
//   dz = dout (y + D u) silu'(z),  dD = sum dy u.
// The forward's state before every tile is read back; the tile is walked forward once more, its kTT states kept in
// registers (kTT x kMc x kSpt of them), and then backward, where a_t is computed again: keeping it too would halve the
// tile. Sums over a channel's states are the forward's transposed reductions; sums over channels (dB, dC) go over
// the lane's channels in registers, over the warp's by exchanges, over the CTA's warps through shared memory, and
// over CTAs by a buffer of one record per CTA that k_sscan_dbc adds in a fixed order (no atomics: the same
// inputs give the same bits).

template <class IO, int NP, bool Z>
struct EndsSmem {  // one warp's
  static constexpr int CH = Shape<NP, kMcBwd<NP>>::CH;
  struct Raw {
    alignas(16) IO rows[Z ? 3 : 2][kTT][CH];  // delta, dout, z
    alignas(16) IO bc[kTT][NP];
  };
  Raw raw[2];
  alignas(16) float dt[kTT][CH];
  alignas(16) float dy[kTT][CH];
  alignas(16) float c[kTT][NP];
};

// Chunk adjoints for a cut time axis: the gradient reaching the state before the chunk's first step from the
// chunk's own outputs (chunks 1 .. nchunk - 1), and the chunk's sum of dt.
template <class IO, int NP, bool Z>
__global__ void __launch_bounds__(32 * kWarps) k_sscan_bwd_ends(const ScanArgs a) {
  using SM = EndsSmem<IO, NP, Z>;
  constexpr int MC = kMcBwd<NP>;
  using S = Shape<NP, MC>;
  constexpr int LPC = S::LPC, CH = S::CH, PC = S::PC, PR = S::PR;
  extern __shared__ __align__(16) unsigned char sm_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPC;
  SM& sm = reinterpret_cast<SM*>(sm_raw)[warp];
  const Place<CH> w(a, warp);
  if (!w.nc) return;
  const int chunk = blockIdx.y + 1, c4 = lane / LPC * MC, n4 = l * kSpt;
  const int64_t t_lo = (int64_t)chunk * a.chunk, t_end = t_lo + a.chunk < a.T ? t_lo + a.chunk : a.T;
  const int64_t t_live = t_end < w.len ? t_end : w.len;
  const int pc = lane % PC * 2, pr = lane / PC;
  const int ntile = t_live > t_lo ? (int)((t_live - t_lo + kTT - 1) / kTT) : 0;
  const int64_t t_at = t_lo + (ntile ? ntile - 1 : 0) * (int64_t)kTT;  // the last tile comes first
  using Rows = Feed<IO, kTT, CH>;
  Rows fd((const IO*)a.delta + w.b * a.d_sb + t_at * a.d_st + w.d0, a.d_st, w.nc, a.vec, lane);
  Rows fo((const IO*)a.dout + w.b * a.o_sb + t_at * a.o_st + w.d0, a.o_st, w.nc, a.vec, lane);
  Rows fz(Z ? (const IO*)a.z + w.b * a.z_sb + t_at * a.z_st + w.d0 : nullptr, a.z_st, w.nc, a.vec, lane);
  Feed<IO, kTT, NP> fc((const IO*)a.Cm + w.b * a.C_sb + w.g * a.C_sg + t_at * a.C_st, a.C_st, a.N, a.vecbc, lane);
  auto fetch = [&](int rows, int s) {
    auto& r = sm.raw[s];
    if (a.vec) {
      fd.vectors(&r.rows[0][0][0], a.d_st, rows, lane);
      fo.vectors(&r.rows[1][0][0], a.o_st, rows, lane);
      if (Z) fz.vectors(&r.rows[Z ? 2 : 0][0][0], a.z_st, rows, lane);
    } else {
      fd.elements(&r.rows[0][0][0], a.d_st, rows, lane);
      fo.elements(&r.rows[1][0][0], a.o_st, rows, lane);
      if (Z) fz.elements(&r.rows[Z ? 2 : 0][0][0], a.z_st, rows, lane);
    }
    if (a.vecbc) fc.vectors(&r.bc[0][0], a.C_st, rows, lane);
    else fc.elements(&r.bc[0][0], a.C_st, rows, lane);
    fd.p -= kTT * a.d_st, fo.p -= kTT * a.o_st, fc.p -= kTT * a.C_st;
    if (Z) fz.p -= kTT * a.z_st;
    cp_commit();
  };
  if (ntile) fetch((int)(t_live - t_at), 0);
  Block<MC> A, q;
  load_A(a, w, c4, n4, A);
  load_state(a, w, nullptr, c4, n4, q);
  const bool c0 = pc < w.nc, c1 = pc + 1 < w.nc;
  const f2 bias = pk(c0 && a.bias ? a.bias[w.d0 + pc] : 0.f, c1 && a.bias ? a.bias[w.d0 + pc + 1] : 0.f);
  f2 sdt = 0;
  int rows = (int)(t_live - t_at);
  for (int it = ntile - 1, s = 0; it >= 0; --it, s ^= 1, rows = kTT) {
    if (it > 0) {
      fetch(kTT, s ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncwarp();
    auto& raw = sm.raw[s];
#pragma unroll
    for (int k = 0; k < kTT; k += PR) {
      const int tt = pr + k;
      f2 x = add2(ld2(&raw.rows[0][tt][pc]), bias), dy = ld2(&raw.rows[1][tt][pc]);
      if (a.softplus) x = softplus_2(x);
      if (tt >= rows) x = 0;
      if (Z) {
        const f2 z = ld2(&raw.rows[Z ? 2 : 0][tt][pc]);
        dy = mul2(dy, mul2(z, sigmoid_2(z)));
      }
      sdt = add2(sdt, x);
      st2(&sm.dt[tt][pc], x);
      st2(&sm.dy[tt][pc], dy);
    }
    widen<IO, NP>(sm.c, &raw.bc[0][0], lane);
    __syncwarp();
#pragma unroll
    for (int tt = kTT - 1; tt >= 0; --tt) {
      const Chans<MC> dt(&sm.dt[tt][c4]), dy(&sm.dy[tt][c4]);
      const States C(&sm.c[tt][n4]);
#pragma unroll
      for (int c = 0; c < MC; ++c)
#pragma unroll
        for (int p = 0; p < kSpt / 2; ++p)
          q.v[c][p] = mul2(ex2_2(mul2(A.v[c][p], dt.v[c])), fma2(C.v[p], dy.v[c], q.v[c][p]));
    }
    __syncwarp();
  }
  const int64_t at = ((int64_t)w.b * a.nchunk + chunk) * a.Dm + w.d0;
  store_rows<NP>(a.part_h + at * NP, w.nc, c4, n4, q);
  const float2 v = up(over_rows<PC>(sdt));
  if (pr == 0 && c0) a.part_dt[at + pc] = v.x;
  if (pr == 0 && c1) a.part_dt[at + pc + 1] = v.y;
}

template <class IO, int NP, bool Z>
struct BwdSmem {
  static constexpr int CH = Shape<NP, kMcBwd<NP>>::CH;
  struct Raw {
    alignas(16) IO rows[Z ? 4 : 3][kTT][CH];  // delta, u, dout, z
    alignas(16) float h[CH][NP];      // the state before the tile
  };
  struct Warp {
    Raw raw[2];
    alignas(16) IO bc[2][kTT][NP];
    alignas(16) float dt[kTT][CH];
    alignas(16) float du[kTT][CH];
    alignas(16) float dy[kTT][CH];
    alignas(16) float b[kTT][NP];
    alignas(16) float c[kTT][NP];
    alignas(16) float y[Z ? 3 : 2][kTT][CH];  // s1, s2, y
  };
  Warp warp[kWarps];
  alignas(16) float red[2][kWarps][kTT][2][NP];  // d B, d C over a warp's channels, two tiles' worth
};

template <class IO, int NP, bool Z>
__global__ void __launch_bounds__(32 * kWarps, kBwdCtas) k_sscan_bwd(const ScanArgs a) {
  using SM = BwdSmem<IO, NP, Z>;
  constexpr int MC = kMcBwd<NP>;
  using S = Shape<NP, MC>;
  constexpr int LPC = S::LPC, CH = S::CH, PC = S::PC, PR = S::PR, SY = S::SY, SB = S::SB, Q = S::Q;
  extern __shared__ __align__(16) unsigned char sm_raw[];
  SM& all = *reinterpret_cast<SM*>(sm_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPC, qd = lane / LPC;
  auto& sm = all.warp[warp];
  const Place<CH> w(a, warp);  // a warp without channels walks along with zeros: the CTA adds over its warps
  const int chunk = blockIdx.y, c4 = qd * MC, n4 = l * kSpt;
  const int64_t t_lo = (int64_t)chunk * a.chunk, t_end = t_lo + a.chunk < a.T ? t_lo + a.chunk : a.T;
  const int64_t t_live = t_end < w.len ? t_end : w.len;
  const int64_t nblk = (a.T + kTT - 1) / kTT;
  const int pc = lane % PC * 2, pr = lane / PC;
  const int ntile = t_live > t_lo ? (int)((t_live - t_lo + kTT - 1) / kTT) : 0;
  const int64_t t_at = t_lo + (ntile ? ntile - 1 : 0) * (int64_t)kTT;  // the last tile comes first
  using Rows = Feed<IO, kTT, CH>;
  using Cols = Feed<IO, kTT, NP>;
  Rows fd((const IO*)a.delta + w.b * a.d_sb + t_at * a.d_st + w.d0, a.d_st, w.nc, a.vec, lane);
  Rows fu((const IO*)a.u + w.b * a.u_sb + t_at * a.u_st + w.d0, a.u_st, w.nc, a.vec, lane);
  Rows fo((const IO*)a.dout + w.b * a.o_sb + t_at * a.o_st + w.d0, a.o_st, w.nc, a.vec, lane);
  Rows fz(Z ? (const IO*)a.z + w.b * a.z_sb + t_at * a.z_st + w.d0 : nullptr, a.z_st, w.nc, a.vec, lane);
  Cols fb((const IO*)a.Bm + w.b * a.B_sb + w.g * a.B_sg + t_at * a.B_st, a.B_st, a.N, a.vecbc, lane);
  Cols fc((const IO*)a.Cm + w.b * a.C_sb + w.g * a.C_sg + t_at * a.C_st, a.C_st, a.N, a.vecbc, lane);
  Feed<float, CH, NP> fh(a.hsave + ((w.b * nblk + t_at / kTT) * a.Dm + w.d0) * NP, NP, NP, 1, lane);
  auto fetch = [&](int rows, int s) {
    auto& r = sm.raw[s];
    if (a.vec) {
      fd.vectors(&r.rows[0][0][0], a.d_st, rows, lane);
      fu.vectors(&r.rows[1][0][0], a.u_st, rows, lane);
      fo.vectors(&r.rows[2][0][0], a.o_st, rows, lane);
      if (Z) fz.vectors(&r.rows[Z ? 3 : 0][0][0], a.z_st, rows, lane);
    } else {
      fd.elements(&r.rows[0][0][0], a.d_st, rows, lane);
      fu.elements(&r.rows[1][0][0], a.u_st, rows, lane);
      fo.elements(&r.rows[2][0][0], a.o_st, rows, lane);
      if (Z) fz.elements(&r.rows[Z ? 3 : 0][0][0], a.z_st, rows, lane);
    }
    if (a.vecbc) {
      fb.vectors(&sm.bc[0][0][0], a.B_st, rows, lane);
      fc.vectors(&sm.bc[1][0][0], a.C_st, rows, lane);
    } else {
      fb.elements(&sm.bc[0][0][0], a.B_st, rows, lane);
      fc.elements(&sm.bc[1][0][0], a.C_st, rows, lane);
    }
    fh.vectors(&r.h[0][0], NP, w.nc, lane);
    fd.p -= kTT * a.d_st, fu.p -= kTT * a.u_st, fo.p -= kTT * a.o_st, fb.p -= kTT * a.B_st, fc.p -= kTT * a.C_st;
    if (Z) fz.p -= kTT * a.z_st;
    fh.p -= (int64_t)a.Dm * NP;
    cp_commit();
  };
  if (ntile) fetch((int)(t_live - t_at), 0);

  Block<MC> A, q, dA;
  load_A(a, w, c4, n4, A);
  if (a.nchunk > 1)
    load_rows<NP>(a.part_h + (((int64_t)w.b * a.nchunk + chunk) * a.Dm + w.d0) * NP, w.nc, c4, n4, q);
  else
    load_state(a, w, a.dhT, c4, n4, q);
  load_state(a, w, nullptr, c4, n4, dA);
  const bool c0 = pc < w.nc, c1 = pc + 1 < w.nc, whole = a.pair && w.nc == CH;
  const f2 bias = pk(c0 && a.bias ? a.bias[w.d0 + pc] : 0.f, c1 && a.bias ? a.bias[w.d0 + pc + 1] : 0.f);
  const f2 skip = pk(c0 && a.D ? a.D[w.d0 + pc] : 0.f, c1 && a.D ? a.D[w.d0 + pc + 1] : 0.f);
  f2 accD = 0, accb = 0;
  float* dbc = a.dbc + ((int64_t)w.tile * a.Bsz + w.b) * a.T * 2 * NP;

  // rows past the length: zero gradients
  const int64_t dead = t_lo > w.len ? t_lo : w.len;
  for (int64_t t = dead + pr; t < t_end; t += PR) {
    const int64_t at = (w.b * a.T + t) * a.Dm + w.d0 + pc;
    store2((IO*)a.du + at, 0, whole, c0, c1);
    store2((IO*)a.ddelta + at, 0, whole, c0, c1);
    if (Z) store2((IO*)a.dz + at, 0, whole, c0, c1);
  }
  for (int64_t i = threadIdx.x; i < (t_end - dead) * 2 * NP; i += 32 * kWarps) dbc[dead * 2 * NP + i] = 0.f;

  int64_t at = (w.b * a.T + t_at + pr) * a.Dm + w.d0 + pc;  // the lane's place in the row outputs
  dbc += t_at * 2 * NP;
  int rows = (int)(t_live - t_at);
  for (int it = ntile - 1, s = 0; it >= 0; --it, s ^= 1, rows = kTT) {
    cp_wait<0>();
    __syncwarp();
    auto& raw = sm.raw[s];
#pragma unroll
    for (int k = 0; k < kTT; k += PR) {
      const int tt = pr + k;
      f2 x = add2(ld2(&raw.rows[0][tt][pc]), bias), dy = ld2(&raw.rows[2][tt][pc]);
      if (a.softplus) x = softplus_2(x);
      if (tt >= rows) x = 0;
      if (Z) {
        const f2 z = ld2(&raw.rows[Z ? 3 : 0][tt][pc]);
        dy = mul2(dy, mul2(z, sigmoid_2(z)));
      }
      st2(&sm.dt[tt][pc], x);
      st2(&sm.du[tt][pc], mul2(x, ld2(&raw.rows[1][tt][pc])));
      st2(&sm.dy[tt][pc], dy);
    }
    widen<IO, NP>(sm.b, &sm.bc[0][0][0], lane);
    widen<IO, NP>(sm.c, &sm.bc[1][0][0], lane);
    __syncwarp();
    if (it > 0) fetch(kTT, s ^ 1);  // B and C have been taken out of their single buffer

    // sums over a channel's lanes of SY steps from ts, to rows of y
    auto put_row = [&](float* p, int ts, float (*dst)[CH]) {
      reduce_part<SY * MC, LPC, 1>(p, lane);
      constexpr int R = SY * MC / LPC;
#pragma unroll
      for (int r = 0; r < R; ++r) dst[ts + l * R / MC][c4 + l * R % MC + r] = p[r];
    };
    // sums over the warp's channel groups of SB steps from ts: d B (part 0), d C (part 1)
    auto put_bc = [&](f2* p, int ts, int part) {
      reduce_pairs<SB * kSpt / 2, Q, LPC>(p, lane);
      constexpr int R = SB * kSpt / Q;
      float* o = &all.red[s][warp][ts + qd * R / kSpt][part][n4 + qd * R % kSpt];
      if (R == 1) o[0] = up(p[0]).x;
      else st2(o, p[0]);
      static_assert(R <= 2, "one pair at most");
    };

    Block<MC> hb[kTT];  // the state before each step
    load_rows<NP>(&raw.h[0][0], CH, c4, n4, hb[0]);
    {
      float py[SY * MC];
      f2 pb[SB * kSpt / 2];
#pragma unroll
      for (int tt = 0; tt < kTT; ++tt) {
        Block<MC> h;
        advance(h, hb[tt], A, Chans<MC>(&sm.dt[tt][c4]), Chans<MC>(&sm.du[tt][c4]), States(&sm.b[tt][n4]));
        if (tt + 1 < kTT) hb[tt + 1 < kTT ? tt + 1 : 0] = h;
        if (Z) {
          dot(py + tt % SY * MC, h, States(&sm.c[tt][n4]));
          if (tt % SY == SY - 1) put_row(py, tt + 1 - SY, sm.y[Z ? 2 : 0]);
        }
        const Chans<MC> dy(&sm.dy[tt][c4]);
#pragma unroll
        for (int p = 0; p < kSpt / 2; ++p) {
          f2 v = mul2(dy.v[0], h.v[0][p]);
#pragma unroll
          for (int c = 1; c < MC; ++c) v = fma2(dy.v[c], h.v[c][p], v);
          pb[tt % SB * (kSpt / 2) + p] = v;
        }
        if (tt % SB == SB - 1) put_bc(pb, tt + 1 - SB, 1);
      }
    }
    {
      float p1[SY * MC], p2[SY * MC];
      f2 pb[SB * kSpt / 2];
#pragma unroll
      for (int tt = kTT - 1; tt >= 0; --tt) {
        const Chans<MC> dt(&sm.dt[tt][c4]), du(&sm.du[tt][c4]), dy(&sm.dy[tt][c4]);
        const States B(&sm.b[tt][n4]), C(&sm.c[tt][n4]);
#pragma unroll
        for (int c = 0; c < MC; ++c) {
          f2 x1, x2;
#pragma unroll
          for (int p = 0; p < kSpt / 2; ++p) {
            const f2 gg = fma2(C.v[p], dy.v[c], q.v[c][p]);
            q.v[c][p] = mul2(ex2_2(mul2(A.v[c][p], dt.v[c])), gg);
            const f2 wv = mul2(q.v[c][p], hb[tt].v[c][p]);  // g a h_{t-1}
            x1 = p ? fma2(gg, B.v[p], x1) : mul2(gg, B.v[p]);
            x2 = p ? fma2(wv, A.v[c][p], x2) : mul2(wv, A.v[c][p]);  // in units of log2(e)
            dA.v[c][p] = fma2(wv, dt.v[c], dA.v[c][p]);
            f2& vb = pb[tt % SB * (kSpt / 2) + p];
            vb = c ? fma2(gg, du.v[c], vb) : mul2(gg, du.v[c]);
          }
          const float2 v1 = up(x1), v2 = up(x2);
          p1[tt % SY * MC + c] = v1.x + v1.y;
          p2[tt % SY * MC + c] = v2.x + v2.y;
        }
        if (tt % SY == 0) {
          put_row(p1, tt, sm.y[0]);
          put_row(p2, tt, sm.y[1]);
        }
        if (tt % SB == 0) put_bc(pb, tt, 0);
      }
    }
    __syncwarp();

    // the tile's rows: du, ddelta, dz; their share of d D and d bias
    auto rows_out = [&](auto whole_tile_) {
      constexpr bool whole_tile = decltype(whole_tile_)::value;
#pragma unroll
      for (int k = 0; k < kTT; k += PR) {
        const int tt = pr + k;
        const f2 u = ld2(&raw.rows[1][tt][pc]), dy = ld2(&sm.dy[tt][pc]), s1 = ld2(&sm.y[0][tt][pc]);
        const f2 du = fma2(ld2(&sm.dt[tt][pc]), s1, mul2(skip, dy));
        f2 dd = fma2(u, s1, mul2(ld2(&sm.y[1][tt][pc]), both(0.6931471805599453f)));
        if (a.softplus) dd = mul2(dd, sigmoid_2(add2(ld2(&raw.rows[0][tt][pc]), bias)));
        f2 dz = 0;
        if (Z) {
          const f2 z = ld2(&raw.rows[Z ? 3 : 0][tt][pc]), sg = sigmoid_2(z);
          const f2 y = fma2(skip, u, ld2(&sm.y[Z ? 2 : 0][tt][pc]));
          // silu'(z) = sg (1 + z (1 - sg))
          dz = mul2(mul2(ld2(&raw.rows[2][tt][pc]), y), mul2(sg, fma2(z, fma2(sg, both(-1.f), both(1.f)), both(1.f))));
        }
        const int64_t o = at + k * (int64_t)a.Dm;
        if (whole_tile || tt < rows) {
          accD = fma2(dy, u, accD);
          accb = add2(accb, dd);
          if (whole_tile) {
            st2((IO*)a.du + o, du);
            st2((IO*)a.ddelta + o, dd);
            if (Z) st2((IO*)a.dz + o, dz);
          } else {
            store2((IO*)a.du + o, du, whole, c0, c1);
            store2((IO*)a.ddelta + o, dd, whole, c0, c1);
            if (Z) store2((IO*)a.dz + o, dz, whole, c0, c1);
          }
        }
      }
    };
    if (whole && rows >= kTT) rows_out(std::true_type());
    else rows_out(std::false_type());
    at -= kTT * (int64_t)a.Dm;
    __syncthreads();  // one a tile: the records of the other buffer are written next
#pragma unroll
    for (int k = 0; k < kTT * 2 * NP / 2; k += 32 * kWarps) {
      const int i = (k + threadIdx.x) * 2;
      if (i < (rows < kTT ? rows : kTT) * 2 * NP) {
        f2 v = 0;
#pragma unroll
        for (int j = 0; j < kWarps; ++j) v = add2(v, ld2(&all.red[s][j][0][0][0] + i));
        st2(dbc + i, v);
      }
    }
    dbc -= kTT * 2 * NP;
  }

  const int64_t part = (int64_t)w.b * a.nchunk + chunk;
  store_rows<NP>(a.part_dA + (part * a.Dm + w.d0) * NP, w.nc, c4, n4, dA);
  if (chunk == 0 && a.dh0) store_state(a, w, a.dh0, c4, n4, q);
  const float2 vD = up(over_rows<PC>(accD)), vb = up(over_rows<PC>(accb));
  if (pr == 0) {
    float* o = a.part_dD + part * 2 * a.Dm + w.d0 + pc;
    if (c0) o[0] = vD.x, o[a.Dm] = vb.x;
    if (c1) o[1] = vD.y, o[a.Dm + 1] = vb.y;
  }
}

// d B, d C: the sum of the channel tiles' records, in tile order. One thread per 4 states; rows past the
// length hold zeros. grid: `blocks` for each group.
template <class IO, int NP>
__global__ void __launch_bounds__(256) k_sscan_dbc(const float* dbc, IO* dB, IO* dC, int64_t rows, int N, int G,
                                                   int tiles, unsigned blocks) {
  const int g = blockIdx.x / blocks;
  const int64_t i = ((int64_t)(blockIdx.x - g * blocks) * 256 + threadIdx.x) * 4;  // over the group's [rows, 2, NP]
  if (i >= rows * 2 * NP) return;
  const float* p = dbc + (int64_t)g * tiles * rows * 2 * NP + i;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = 0; k < tiles; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)k * rows * 2 * NP);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const int64_t row = i / (2 * NP);
  const int r = (int)(i - row * 2 * NP), n = r % NP;
  IO* o = (r < NP ? dB : dC) + (row * G + g) * N + n;
  if (n < N) from_f(o[0], s.x);
  if (n + 1 < N) from_f(o[1], s.y);
  if (n + 2 < N) from_f(o[2], s.z);
  if (n + 3 < N) from_f(o[3], s.w);
}

// d A [Dm, N], d D, d bias [Dm]: the sum over batch rows and chunks, in order.
__global__ void __launch_bounds__(256) k_sscan_dA(const float* part_dA, const float* part_dD, float* dA, float* dD,
                                                  float* dbias, int parts, int Dm, int N, int NP) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t na = (int64_t)Dm * NP;
  if (i < na) {
    const int n = (int)(i % NP);
    if (n >= N) return;
    float s = 0.f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) s += part_dA[p * na + i];
    dA[i / NP * N + n] = s;
  } else if (i < na + 2 * (int64_t)Dm) {
    const int64_t j = i - na;
    float s = 0.f;
    for (int p = 0; p < parts; ++p) s += part_dD[p * 2 * (int64_t)Dm + j];
    float* o = j < Dm ? dD : dbias;
    if (o) o[j < Dm ? j : j - Dm] = s;
  }
}

}  // namespace ss
}  // namespace atlas
