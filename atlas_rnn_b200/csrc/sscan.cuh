// Selective state space scan: per batch row, channel d and state n
//   dt_t = softplus(delta_t + bias) (or delta_t + bias),  a_t = exp(dt_t A[d,n]),
//   h_t  = a_t h_{t-1} + dt_t u_t B_t[n],  y_t = sum_n C_t[n] h_t + D u_t,  out_t = y_t silu(z_t),
// and its backward. The scalar-gated scans of scan_op.cuh share one gate over the whole state; here
// every (channel, state) pair has its own, so the exponentials, one per (token, channel, state), set
// the floor: 16 per cycle and SM on the special-function unit, against about 20 bytes of traffic
// per (token, channel).
//
// Layout of the work: a channel's states lie across LPC = NP / SPT lanes, SPT states a lane (NP: the
// state count padded to a power of two with A = B = C = 0 columns, whose states stay 0). A CTA owns
// kThr / LPC neighbouring channels and walks the time axis in tiles of kTT steps: the tile's rows
// are read once, coalesced, one tile ahead of their use; dt and dt u go through shared memory
// as fp32, B and C too (shared by all channels of the tile); the walk itself runs in
// registers; the sums over a channel's lanes are transposed reductions over LPC steps at
// a time (LPC - 1 shuffles give LPC steps' sums, one per lane). Lengths: a step at or past its row's
// length has dt = 0 (a = 1, no input) and writes 0.
//
// When the rows and channels do not fill the machine, the time axis is cut into chunks: a first
// pass leaves each chunk's own end state (from zero) and its sum of dt, the second starts
// every chunk from h = sum over earlier chunks, each decayed by exp(A sum dt). That pays the
// exponentials twice.
#pragma once
#include "row_ops.cuh"

namespace atlas {
namespace ss {

constexpr int kTT = 32;       // steps per tile
constexpr int kSaveSteps = 16;  // training: the state before every 16th step is kept for the backward

struct ScanArgs {
  const void *u, *delta, *z, *Bm, *Cm, *dout;
  int64_t u_sb, u_st, d_sb, d_st, z_sb, z_st, o_sb, o_st;  // element strides (batch, step); channels are dense
  int64_t B_sb, B_st, B_sg, C_sb, C_st, C_sg;              // (batch, step, group); states are dense
  const float *A, *D, *bias, *h0;
  const int* len;
  void* out;       // [B, T, Dm]
  float* hT;       // [B, Dm, N]
  float* hsave;    // [B, ceil(T / kSaveSteps), Dm, NP]
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
  int vecbc; // B and C allow 4-element accesses
};

// ---- forward --------------------------------------------------------------
constexpr int kFwdThr = 128;

// Row tile of a CTA: R rows of CH channels; the thread's elements are W neighbours of one or more rows.
template <class IO, int CH, int THR, int ROWS>
struct RowTile {
  static constexpr int kEach = ROWS * CH / THR;                 // elements per thread
  static constexpr int kMax = 16 / (int)sizeof(IO);
  static constexpr int W = kEach < kMax ? (kEach < CH ? kEach : CH) : (kMax < CH ? kMax : CH);
  static constexpr int kVecs = kEach / W;
  static constexpr int kCols = CH / W, kRowStep = THR / kCols;
  static_assert(kEach >= 1 && kVecs * W == kEach && kCols * W == CH && kRowStep * kVecs == ROWS, "row tile");
};

// grid (batch x groups x channel tiles, chunks). ENDS: only the chunk's end state and sum of dt.
template <class IO, int NP, int SPT, bool ENDS>
__global__ void __launch_bounds__(kFwdThr) k_sscan_fwd(const ScanArgs a) {
  constexpr int LPC = NP / SPT, CH = kFwdThr / LPC, CPW = 32 / LPC, YS = CH + CPW, P2 = SPT / 2;
  using RT = RowTile<IO, CH, kFwdThr, kTT>;
  constexpr int W = RT::W, NV = RT::kVecs;
  constexpr int BU = kTT * NP / 4 / kFwdThr > 0 ? kTT * NP / 4 / kFwdThr : 1;  // 4-state units of B per thread
  __shared__ __align__(16) float2 s_dt[kTT][CH];
  __shared__ __align__(16) float s_b[kTT][NP];
  __shared__ __align__(16) float s_c[ENDS ? 1 : kTT][NP];
  __shared__ __align__(16) float s_y[ENDS ? 1 : kTT][YS];
  const int tid = threadIdx.x, lane = tid & 31, l = lane % LPC, ch = tid / LPC;
  const int Dg = a.Dm / a.G, tiles = (Dg + CH - 1) / CH;
  const int b = blockIdx.x / (tiles * a.G), gt = blockIdx.x - b * tiles * a.G;
  const int g = gt / tiles, cbase = (gt - g * tiles) * CH;  // channel tile inside its group
  const int chunk = blockIdx.y;
  const int64_t t_lo = (int64_t)chunk * a.chunk, t_hi = t_lo + a.chunk < a.T ? t_lo + a.chunk : a.T;
  const int64_t len = row_len(a.len, b, a.T);
  const int nc = Dg - cbase < CH ? Dg - cbase : CH;  // channels of this tile
  const int64_t d0 = (int64_t)g * Dg + cbase;
  const IO* up_ = (const IO*)a.u + b * a.u_sb + d0;
  const IO* dp_ = (const IO*)a.delta + b * a.d_sb + d0;
  const IO* zp_ = a.z ? (const IO*)a.z + b * a.z_sb + d0 : nullptr;
  const IO* bp_ = (const IO*)a.Bm + b * a.B_sb + g * a.B_sg;
  const IO* cp_ = (const IO*)a.Cm + b * a.C_sb + g * a.C_sg;
  const int rcol = (tid % RT::kCols) * W, rrow = tid / RT::kCols;

  // this lane's states: A in units of log2, the state the chunk starts from
  const bool mine = ch < nc;
  f2 A2[P2], h[P2];
  {
    float av[SPT], hv[SPT];
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      const int n = l * SPT + i;
      av[i] = mine && n < a.N ? a.A[(d0 + ch) * a.N + n] * kLog2e : 0.f;
      hv[i] = !ENDS && mine && n < a.N && a.h0 ? a.h0[((int64_t)b * a.Dm + d0 + ch) * a.N + n] : 0.f;
    }
    if (!ENDS && mine)
      for (int c = 0; c < chunk; ++c) {
        const int64_t at = ((int64_t)b * a.nchunk + c) * a.Dm + d0 + ch;
        const float sdt = a.part_dt[at];
#pragma unroll
        for (int i = 0; i < SPT; ++i) hv[i] = fmaf(ex2(av[i] * sdt), hv[i], a.part_h[at * NP + l * SPT + i]);
      }
#pragma unroll
    for (int i = 0; i < P2; ++i) A2[i] = pk(av[2 * i], av[2 * i + 1]), h[i] = pk(hv[2 * i], hv[2 * i + 1]);
  }
  float bias[W], Dv[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const bool ok = rcol + i < nc;
    bias[i] = ok && a.bias ? a.bias[d0 + rcol + i] : 0.f;
    Dv[i] = ok && a.D ? a.D[d0 + rcol + i] : 0.f;
  }
  float sdt[W];
#pragma unroll
  for (int i = 0; i < W; ++i) sdt[i] = 0.f;

  Vec<IO, W> ru[NV], rd[NV], rz[NV];
  Vec<IO, 4> rb[BU], rc[BU];
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t t = t0 + rrow + v * RT::kRowStep;
      if (t < t_hi && t < len) {
        ru[v] = load_row<IO, W>(up_ + t * a.u_st, rcol, nc, a.vec);
        rd[v] = load_row<IO, W>(dp_ + t * a.d_st, rcol, nc, a.vec);
        if (!ENDS && zp_) rz[v] = load_row<IO, W>(zp_ + t * a.z_st, rcol, nc, a.vec);
      } else {
        ru[v] = rd[v] = rz[v] = zero_row<IO, W>();
      }
    }
#pragma unroll
    for (int v = 0; v < BU; ++v) {
      const int at = tid + v * kFwdThr, tt = at / (NP / 4), n = (at % (NP / 4)) * 4;
      rb[v] = rc[v] = zero_row<IO, 4>();
      if (tt < kTT && t0 + tt < t_hi && t0 + tt < len) {
        rb[v] = load_row<IO, 4>(bp_ + (t0 + tt) * a.B_st, n, a.N, a.vecbc);
        if (!ENDS) rc[v] = load_row<IO, 4>(cp_ + (t0 + tt) * a.C_st, n, a.N, a.vecbc);
      }
    }
  };
  const int64_t nblk = (a.T + kSaveSteps - 1) / kSaveSteps;

  fetch(t_lo);
  for (int64_t t0 = t_lo; t0 < t_hi; t0 += kTT) {
    if (t0 >= len) {  // nothing but zeros from here on (the whole CTA: len is the row's)
      if (!ENDS) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int64_t t = t0 + rrow + v * RT::kRowStep;
          if (t < t_hi)
            store_row<IO, W>((IO*)a.out + (b * a.T + t) * a.Dm + d0, rcol, nc, a.vec, zero_row<IO, W>());
        }
        continue;
      }
      break;
    }
    // dt, dt u, B, C of the tile; the raw rows of u and z stay for the epilogue
    Vec<IO, W> cu[NV], cz[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int tt = rrow + v * RT::kRowStep;
      const bool live = t0 + tt < t_hi && t0 + tt < len;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float x = to_f(rd[v].v[i]) + bias[i];
        if (a.softplus) x = softplus(x);
        if (!live) x = 0.f;
        sdt[i] += x;
        s_dt[tt][rcol + i] = make_float2(x, x * to_f(ru[v].v[i]));
      }
      cu[v] = ru[v];
      cz[v] = rz[v];
    }
#pragma unroll
    for (int v = 0; v < BU; ++v) {
      const int at = tid + v * kFwdThr, tt = at / (NP / 4), n = (at % (NP / 4)) * 4;
      if (tt < kTT) {
        *reinterpret_cast<float4*>(&s_b[tt][n]) =
            make_float4(to_f(rb[v].v[0]), to_f(rb[v].v[1]), to_f(rb[v].v[2]), to_f(rb[v].v[3]));
        if (!ENDS)
          *reinterpret_cast<float4*>(&s_c[tt][n]) =
              make_float4(to_f(rc[v].v[0]), to_f(rc[v].v[1]), to_f(rc[v].v[2]), to_f(rc[v].v[3]));
      }
    }
    __syncthreads();
    if (t0 + kTT < t_hi) fetch(t0 + kTT);

#pragma unroll 1
    for (int tg = 0; tg < kTT; tg += LPC) {
      if (!ENDS && a.hsave && tg % kSaveSteps == 0 && mine && t0 + tg < a.T) {
        float* hs = a.hsave + ((b * nblk + (t0 + tg) / kSaveSteps) * a.Dm + d0 + ch) * NP + l * SPT;
#pragma unroll
        for (int i = 0; i < P2; ++i) reinterpret_cast<float2*>(hs)[i] = up(h[i]);
      }
      float p[LPC];
#pragma unroll
      for (int j = 0; j < LPC; ++j) {
        const int tt = tg + j;
        if (!ENDS && LPC > kSaveSteps && j == kSaveSteps && a.hsave && mine && t0 + tt < a.T) {
          float* hs = a.hsave + ((b * nblk + (t0 + tt) / kSaveSteps) * a.Dm + d0 + ch) * NP + l * SPT;
#pragma unroll
          for (int i = 0; i < P2; ++i) reinterpret_cast<float2*>(hs)[i] = up(h[i]);
        }
        const float2 q = s_dt[tt][ch];
        const f2 dt2 = pk(q.x, q.x), du2 = pk(q.y, q.y);
        const f2* Bv = reinterpret_cast<const f2*>(&s_b[tt][l * SPT]);
        const f2* Cv = reinterpret_cast<const f2*>(&s_c[ENDS ? 0 : tt][l * SPT]);
        f2 acc = 0;
#pragma unroll
        for (int i = 0; i < P2; ++i) {
          h[i] = fma2(ex2_2(mul2(A2[i], dt2)), h[i], mul2(du2, Bv[i]));
          if (!ENDS) acc = i == 0 ? mul2(Cv[i], h[i]) : fma2(Cv[i], h[i], acc);
        }
        if (!ENDS) {
          const float2 s = up(acc);
          p[j] = s.x + s.y;
        }
      }
      if (!ENDS) {
        reduce_scatter<LPC, 1>(p, lane);
        s_y[tg + l][ch] = p[0];
      }
    }
    __syncthreads();
    if (!ENDS) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int tt = rrow + v * RT::kRowStep;
        if (t0 + tt >= t_hi) continue;
        const bool live = t0 + tt < len;
        Vec<IO, W> o;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          float y = fmaf(Dv[i], to_f(cu[v].v[i]), s_y[tt][rcol + i]);
          if (zp_) {
            const float zz = to_f(cz[v].v[i]);
            y *= zz * sigmoid(zz);
          }
          from_f(o.v[i], live ? y : 0.f);
        }
        store_row<IO, W>((IO*)a.out + (b * a.T + t0 + tt) * a.Dm + d0, rcol, nc, a.vec, o);
      }
    }
  }
  if (ENDS) {
    if (mine) {
      float* ph = a.part_h + (((int64_t)b * a.nchunk + chunk) * a.Dm + d0 + ch) * NP + l * SPT;
#pragma unroll
      for (int i = 0; i < P2; ++i) reinterpret_cast<float2*>(ph)[i] = up(h[i]);
    }
    // the chunk's sum of dt per channel, over the threads that share its columns
    __syncthreads();
    float* red = reinterpret_cast<float*>(s_dt);  // [kRowStep][CH]
#pragma unroll
    for (int i = 0; i < W; ++i) red[rrow * CH + rcol + i] = sdt[i];
    __syncthreads();
    if (tid < nc) {
      float s = 0.f;
      for (int r = 0; r < RT::kRowStep; ++r) s += red[r * CH + tid];
      a.part_dt[((int64_t)b * a.nchunk + chunk) * a.Dm + d0 + tid] = s;
    }
  } else if (mine && chunk == a.nchunk - 1) {
#pragma unroll
    for (int i = 0; i < P2; ++i) {
      const float2 v = up(h[i]);
      const int n = l * SPT + 2 * i;
      float* o = a.hT + ((int64_t)b * a.Dm + d0 + ch) * a.N + n;
      if (n < a.N) o[0] = v.x;
      if (n + 1 < a.N) o[1] = v.y;
    }
  }
}

// ---- one token ------------------------------------------------------------
// T = 1 without a backward: a thread takes 4 neighbouring states (one 16-byte read and write of the
// state, which is the traffic), LPC = NP / 4 lanes a channel.
constexpr int kStepThr = 128;
template <class IO, int NP>
__global__ void __launch_bounds__(kStepThr) k_sscan_step(const ScanArgs a, int vec4) {
  constexpr int LPC = NP / 4;
  const int64_t at = (int64_t)blockIdx.x * (kStepThr / LPC) + threadIdx.x / LPC;  // b * Dm + d
  const int l = threadIdx.x % LPC;
  const bool mine = at < (int64_t)a.Bsz * a.Dm;
  const int b = mine ? (int)(at / a.Dm) : 0, d = mine ? (int)(at % a.Dm) : 0, g = d / (a.Dm / a.G);
  const bool live = mine && row_len(a.len, b, 1) > 0;
  float Av[4] = {0.f, 0.f, 0.f, 0.f}, hv[4] = {0.f, 0.f, 0.f, 0.f};
  if (mine) {
    const float *Ap = a.A + (int64_t)d * a.N + l * 4, *hp = a.h0 ? a.h0 + at * a.N + l * 4 : nullptr;
    if (vec4) {
      if (l * 4 < a.N) {
        const float4 x = *reinterpret_cast<const float4*>(Ap);
        Av[0] = x.x, Av[1] = x.y, Av[2] = x.z, Av[3] = x.w;
        if (hp) {
          const float4 y = *reinterpret_cast<const float4*>(hp);
          hv[0] = y.x, hv[1] = y.y, hv[2] = y.z, hv[3] = y.w;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (l * 4 + i < a.N) {
          Av[i] = Ap[i];
          if (hp) hv[i] = hp[i];
        }
    }
  }
  float dt = 0.f, uu = 0.f, zz = 0.f;
  Vec<IO, 4> Bv = zero_row<IO, 4>(), Cv = Bv;
  if (live) {
    uu = to_f(((const IO*)a.u)[b * a.u_sb + d]);
    dt = to_f(((const IO*)a.delta)[b * a.d_sb + d]) + (a.bias ? a.bias[d] : 0.f);
    if (a.z) zz = to_f(((const IO*)a.z)[b * a.z_sb + d]);
    if (a.softplus) dt = softplus(dt);
    Bv = load_row<IO, 4>((const IO*)a.Bm + b * a.B_sb + g * a.B_sg, l * 4, a.N, a.vecbc);
    Cv = load_row<IO, 4>((const IO*)a.Cm + b * a.C_sb + g * a.C_sg, l * 4, a.N, a.vecbc);
  }
  float y = 0.f;
  const float dl = dt * kLog2e, du = dt * uu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hv[i] = fmaf(ex2(Av[i] * dl), hv[i], du * to_f(Bv.v[i]));
    y = fmaf(to_f(Cv.v[i]), hv[i], y);
  }
#pragma unroll
  for (int o = LPC / 2; o >= 1; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (!mine) return;
  float* ho = a.hT + at * a.N + l * 4;
  if (vec4) {
    if (l * 4 < a.N) *reinterpret_cast<float4*>(ho) = make_float4(hv[0], hv[1], hv[2], hv[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (l * 4 + i < a.N) ho[i] = hv[i];
  }
  if (l == 0) {
    if (a.D) y = fmaf(a.D[d], uu, y);
    if (a.z) y *= zz * sigmoid(zz);
    from_f(((IO*)a.out)[at], live ? y : 0.f);
  }
}

// ---- backward -------------------------------------------------------------
// With dy = dout silu(z) and g_t the gradient reaching h_t:
//   g_t = C_t dy_t + a_{t+1} g_{t+1} (from dhT),  q_t = a_t g_t reaches h_{t-1};
//   dC_t = sum_d dy_t h_t,  dB_t = sum_d g_t dt_t u_t,  s1_t = sum_n g_t B_t,  w = g_t a_t h_{t-1},
//   du = dt s1 + D dy,  d dt = sum_n w A + u s1,  dA = sum_t w dt,  ddelta = d dt sigmoid(delta + bias),
//   dz = dout (y + D u) silu'(z),  dD = sum dy u.
// The forward's state before every 16th step is read back; each block of 16 steps is walked forward once more
// (a_t and a_t h_{t-1} stay in registers: 2 states a lane) and then backward. Sums over a channel's states
// are the forward's transposed reductions; sums over channels (dB, dC) go over the warp's
// channels by shuffles, over the CTA's warps through shared memory, and over CTAs by a buffer of one
// record per channel tile that k_sscan_dbc adds in a fixed order (no atomics: the same inputs give the same bits).
constexpr int kBwdThr = 256;

// Chunk adjoints for a cut time axis: the gradient reaching the state before the chunk's first step from the
// chunk's own outputs (grid as forward; chunks 1 .. nchunk - 1), and the chunk's sum of dt.
template <class IO, int NP, int SPT>
__global__ void __launch_bounds__(kFwdThr) k_sscan_bwd_ends(const ScanArgs a) {
  constexpr int LPC = NP / SPT, CH = kFwdThr / LPC, P2 = SPT / 2;
  using RT = RowTile<IO, CH, kFwdThr, kTT>;
  constexpr int W = RT::W, NV = RT::kVecs;
  constexpr int BU = kTT * NP / 4 / kFwdThr > 0 ? kTT * NP / 4 / kFwdThr : 1;
  __shared__ __align__(16) float2 s_dt[kTT][CH];  // dt, dy
  __shared__ __align__(16) float s_c[kTT][NP];
  const int tid = threadIdx.x, lane = tid & 31, l = lane % LPC, ch = tid / LPC;
  const int Dg = a.Dm / a.G, tiles = (Dg + CH - 1) / CH;
  const int b = blockIdx.x / (tiles * a.G), gt = blockIdx.x - b * tiles * a.G;
  const int g = gt / tiles, cbase = (gt - g * tiles) * CH;
  const int chunk = blockIdx.y + 1;
  const int64_t t_lo = (int64_t)chunk * a.chunk, t_end = t_lo + a.chunk < a.T ? t_lo + a.chunk : a.T;
  const int64_t len = row_len(a.len, b, a.T), t_hi = t_end < len ? t_end : len;
  const int nc = Dg - cbase < CH ? Dg - cbase : CH;
  const int64_t d0 = (int64_t)g * Dg + cbase;
  const IO* dp_ = (const IO*)a.delta + b * a.d_sb + d0;
  const IO* zp_ = a.z ? (const IO*)a.z + b * a.z_sb + d0 : nullptr;
  const IO* op_ = (const IO*)a.dout + b * a.o_sb + d0;
  const IO* cp_ = (const IO*)a.Cm + b * a.C_sb + g * a.C_sg;
  const int rcol = (tid % RT::kCols) * W, rrow = tid / RT::kCols;
  const bool mine = ch < nc;
  f2 A2[P2], q[P2];
#pragma unroll
  for (int i = 0; i < P2; ++i) {
    const int n = l * SPT + 2 * i;
    const float* Ap = a.A + (d0 + (mine ? ch : 0)) * a.N;
    A2[i] = pk(mine && n < a.N ? Ap[n] * kLog2e : 0.f, mine && n + 1 < a.N ? Ap[n + 1] * kLog2e : 0.f);
    q[i] = 0;
  }
  float bias[W], sdt[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    bias[i] = rcol + i < nc && a.bias ? a.bias[d0 + rcol + i] : 0.f;
    sdt[i] = 0.f;
  }
  const int64_t ntile = t_hi > t_lo ? (t_hi - t_lo + kTT - 1) / kTT : 0;
  for (int64_t it = ntile - 1; it >= 0; --it) {
    const int64_t t0 = t_lo + it * kTT;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int tt = rrow + v * RT::kRowStep;
      const int64_t t = t0 + tt;
      const bool live = t < t_hi;
      Vec<IO, W> rd = zero_row<IO, W>(), ro = rd, rz = rd;
      if (live) {
        rd = load_row<IO, W>(dp_ + t * a.d_st, rcol, nc, a.vec);
        ro = load_row<IO, W>(op_ + t * a.o_st, rcol, nc, a.vec);
        if (zp_) rz = load_row<IO, W>(zp_ + t * a.z_st, rcol, nc, a.vec);
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float x = to_f(rd.v[i]) + bias[i], dy = to_f(ro.v[i]);
        if (a.softplus) x = softplus(x);
        if (!live) x = 0.f;
        if (zp_) dy *= to_f(rz.v[i]) * sigmoid(to_f(rz.v[i]));
        sdt[i] += x;
        s_dt[tt][rcol + i] = make_float2(x, dy);
      }
    }
#pragma unroll
    for (int v = 0; v < BU; ++v) {
      const int at = tid + v * kFwdThr, tt = at / (NP / 4), n = (at % (NP / 4)) * 4;
      if (tt < kTT) {
        Vec<IO, 4> r = zero_row<IO, 4>();
        if (t0 + tt < t_hi) r = load_row<IO, 4>(cp_ + (t0 + tt) * a.C_st, n, a.N, a.vecbc);
        *reinterpret_cast<float4*>(&s_c[tt][n]) = make_float4(to_f(r.v[0]), to_f(r.v[1]), to_f(r.v[2]), to_f(r.v[3]));
      }
    }
    __syncthreads();
#pragma unroll 8
    for (int tt = kTT - 1; tt >= 0; --tt) {
      const float2 e = s_dt[tt][ch];
      const f2 dt2 = pk(e.x, e.x), dy2 = pk(e.y, e.y);
      const f2* Cv = reinterpret_cast<const f2*>(&s_c[tt][l * SPT]);
#pragma unroll
      for (int i = 0; i < P2; ++i) q[i] = mul2(ex2_2(mul2(A2[i], dt2)), fma2(Cv[i], dy2, q[i]));
    }
    __syncthreads();
  }
  if (mine) {
    float* ph = a.part_h + (((int64_t)b * a.nchunk + chunk) * a.Dm + d0 + ch) * NP + l * SPT;
#pragma unroll
    for (int i = 0; i < P2; ++i) reinterpret_cast<float2*>(ph)[i] = up(q[i]);
  }
  __syncthreads();
  float* red = reinterpret_cast<float*>(s_dt);
#pragma unroll
  for (int i = 0; i < W; ++i) red[rrow * CH + rcol + i] = sdt[i];
  __syncthreads();
  if (tid < nc) {
    float s = 0.f;
    for (int r = 0; r < RT::kRowStep; ++r) s += red[r * CH + tid];
    a.part_dt[((int64_t)b * a.nchunk + chunk) * a.Dm + d0 + tid] = s;
  }
}

template <int NP>
struct BwdSmem {
  static constexpr int LPC = NP / 2, CH = kBwdThr / LPC, CPW = 32 / LPC, YS = CH + CPW, WARPS = kBwdThr / 32;
  static constexpr int q = 0;                                // float4 [kTT][CH]: dt, dt u, dy
  static constexpr int b = q + kTT * CH * 16, c = b + kTT * NP * 4;
  static constexpr int y = c + kTT * NP * 4;                 // float [3][kTT][YS]: y, s1, s2
  static constexpr int red = y + 3 * kTT * YS * 4;           // float [WARPS][kTT][2][NP]: d B, d C of a warp's channels
  static constexpr int bytes = red + WARPS * kTT * 2 * NP * 4;
};

template <class IO, int NP>
__global__ void __launch_bounds__(kBwdThr, 2) k_sscan_bwd(const ScanArgs a) {
  using SM = BwdSmem<NP>;
  constexpr int LPC = SM::LPC, CH = SM::CH, CPW = SM::CPW, YS = SM::YS, WARPS = SM::WARPS;
  constexpr int RG = LPC < 16 ? LPC : 16;          // steps per reduction over a channel's lanes
  constexpr int CG = CPW >= 2 ? CPW / 2 : 1;       // steps per reduction over the warp's channels
  using RT = RowTile<IO, CH, kBwdThr, kTT>;
  constexpr int W = RT::W, NV = RT::kVecs;
  constexpr int BU = kTT * NP / 4 / kBwdThr > 0 ? kTT * NP / 4 / kBwdThr : 1;
  extern __shared__ __align__(16) unsigned char sm[];
  float4(*s_q)[CH] = reinterpret_cast<float4(*)[CH]>(sm + SM::q);
  float(*s_b)[NP] = reinterpret_cast<float(*)[NP]>(sm + SM::b);
  float(*s_c)[NP] = reinterpret_cast<float(*)[NP]>(sm + SM::c);
  float(*s_y)[YS] = reinterpret_cast<float(*)[YS]>(sm + SM::y);
  float(*s_1)[YS] = s_y + kTT;
  float(*s_2)[YS] = s_1 + kTT;
  float* s_red = reinterpret_cast<float*>(sm + SM::red);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = lane % LPC, cw = lane / LPC, ch = tid / LPC;
  const int Dg = a.Dm / a.G, tiles = (Dg + CH - 1) / CH;
  const int b = blockIdx.x / (tiles * a.G), gt = blockIdx.x - b * tiles * a.G;
  const int g = gt / tiles, cbase = (gt - g * tiles) * CH;
  const int chunk = blockIdx.y;
  const int64_t t_lo = (int64_t)chunk * a.chunk, t_end = t_lo + a.chunk < a.T ? t_lo + a.chunk : a.T;
  const int64_t len = row_len(a.len, b, a.T), t_hi = t_end < len ? t_end : len;  // live steps: t_lo .. t_hi - 1
  const int nc = Dg - cbase < CH ? Dg - cbase : CH;
  const int64_t d0 = (int64_t)g * Dg + cbase;
  const IO* up_ = (const IO*)a.u + b * a.u_sb + d0;
  const IO* dp_ = (const IO*)a.delta + b * a.d_sb + d0;
  const IO* zp_ = a.z ? (const IO*)a.z + b * a.z_sb + d0 : nullptr;
  const IO* op_ = (const IO*)a.dout + b * a.o_sb + d0;
  const IO* bp_ = (const IO*)a.Bm + b * a.B_sb + g * a.B_sg;
  const IO* cp_ = (const IO*)a.Cm + b * a.C_sb + g * a.C_sg;
  const int rcol = (tid % RT::kCols) * W, rrow = tid / RT::kCols;
  const int64_t nblk = (a.T + kSaveSteps - 1) / kSaveSteps;
  const bool mine = ch < nc;
  const int n0 = l * 2;

  f2 A2, q;
  {
    const int64_t row = (int64_t)b * a.Dm + d0 + (mine ? ch : 0);
    const float* Ap = a.A + (d0 + (mine ? ch : 0)) * a.N;
    const float a0 = mine && n0 < a.N ? Ap[n0] * kLog2e : 0.f, a1 = mine && n0 + 1 < a.N ? Ap[n0 + 1] * kLog2e : 0.f;
    float q0 = 0.f, q1 = 0.f;
    if (mine && a.dhT) {
      if (n0 < a.N) q0 = a.dhT[row * a.N + n0];
      if (n0 + 1 < a.N) q1 = a.dhT[row * a.N + n0 + 1];
    }
    if (mine)
      for (int c = a.nchunk - 1; c > chunk; --c) {
        const int64_t at = ((int64_t)b * a.nchunk + c) * a.Dm + d0 + ch;
        const float sdt = a.part_dt[at];
        const float2 p = *reinterpret_cast<const float2*>(a.part_h + at * NP + n0);
        q0 = fmaf(ex2(a0 * sdt), q0, p.x);
        q1 = fmaf(ex2(a1 * sdt), q1, p.y);
      }
    A2 = pk(a0, a1);
    q = pk(q0, q1);
  }
  float bias[W], Dv[W], accD[W], accb[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const bool ok = rcol + i < nc;
    bias[i] = ok && a.bias ? a.bias[d0 + rcol + i] : 0.f;
    Dv[i] = ok && a.D ? a.D[d0 + rcol + i] : 0.f;
    accD[i] = accb[i] = 0.f;
  }
  f2 dA = 0;

  // rows past the length: zero gradients
  const int64_t dead = t_lo > len ? t_lo : len;
  for (int64_t i = tid; i < (t_end - dead) * nc; i += kBwdThr) {
    const int64_t at = (b * a.T + dead + i / nc) * a.Dm + d0 + i % nc;
    from_f(((IO*)a.du)[at], 0.f);
    from_f(((IO*)a.ddelta)[at], 0.f);
    if (a.dz) from_f(((IO*)a.dz)[at], 0.f);
  }
  if (a.dbc)
    for (int64_t i = tid; i < (t_end - dead) * 2 * NP; i += kBwdThr)
      a.dbc[(((int64_t)gt * a.Bsz + b) * a.T + dead) * 2 * NP + i] = 0.f;

  const int64_t ntile = t_hi > t_lo ? (t_hi - t_lo + kTT - 1) / kTT : 0;
  for (int64_t it = ntile - 1; it >= 0; --it) {
    const int64_t t0 = t_lo + it * kTT;
    Vec<IO, W> ru[NV], rd[NV], rz[NV], ro[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int tt = rrow + v * RT::kRowStep;
      const int64_t t = t0 + tt;
      const bool live = t < t_hi;
      ru[v] = rd[v] = rz[v] = ro[v] = zero_row<IO, W>();
      if (live) {
        ru[v] = load_row<IO, W>(up_ + t * a.u_st, rcol, nc, a.vec);
        rd[v] = load_row<IO, W>(dp_ + t * a.d_st, rcol, nc, a.vec);
        ro[v] = load_row<IO, W>(op_ + t * a.o_st, rcol, nc, a.vec);
        if (zp_) rz[v] = load_row<IO, W>(zp_ + t * a.z_st, rcol, nc, a.vec);
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float x = to_f(rd[v].v[i]) + bias[i], dy = to_f(ro[v].v[i]);
        if (a.softplus) x = softplus(x);
        if (!live) x = 0.f;
        if (zp_) dy *= to_f(rz[v].v[i]) * sigmoid(to_f(rz[v].v[i]));
        s_q[tt][rcol + i] = make_float4(x, x * to_f(ru[v].v[i]), dy, 0.f);
      }
    }
#pragma unroll
    for (int v = 0; v < BU; ++v) {
      const int at = tid + v * kBwdThr, tt = at / (NP / 4), n = (at % (NP / 4)) * 4;
      if (tt < kTT) {
        Vec<IO, 4> r = zero_row<IO, 4>(), s = r;
        if (t0 + tt < t_hi) {
          r = load_row<IO, 4>(bp_ + (t0 + tt) * a.B_st, n, a.N, a.vecbc);
          s = load_row<IO, 4>(cp_ + (t0 + tt) * a.C_st, n, a.N, a.vecbc);
        }
        *reinterpret_cast<float4*>(&s_b[tt][n]) = make_float4(to_f(r.v[0]), to_f(r.v[1]), to_f(r.v[2]), to_f(r.v[3]));
        *reinterpret_cast<float4*>(&s_c[tt][n]) = make_float4(to_f(s.v[0]), to_f(s.v[1]), to_f(s.v[2]), to_f(s.v[3]));
      }
    }
    __syncthreads();

    // d B (part 0) and d C (part 1) of step tt over the warp's channels
    auto put = [&](float* v, int tt, int part) {  // v: CG steps x 2 states, ending at step tt + CG - 1
      if (CPW >= 2) {
        reduce_scatter<CPW >= 2 ? CPW : 2, LPC>(v, lane);
        s_red[((warp * kTT + tt + cw / 2) * 2 + part) * NP + n0 + (cw & 1)] = v[0];
      } else {
        s_red[((warp * kTT + tt) * 2 + part) * NP + n0] = v[0];
        s_red[((warp * kTT + tt) * 2 + part) * NP + n0 + 1] = v[1];
      }
    };
    auto put_row = [&](float* v, int tt, float (*dst)[YS]) {  // RG steps from tt
      reduce_scatter<RG, 1>(v, lane);
      float r = v[0];
      if (LPC > RG) r += __shfl_xor_sync(0xffffffffu, r, 16);
      if (l < RG) dst[tt + l][ch] = r;
    };

#pragma unroll 1
    for (int blk = kTT / kSaveSteps - 1; blk >= 0; --blk) {
      const int tb = blk * kSaveSteps;
      f2 aa[kSaveSteps], ah[kSaveSteps];
      f2 h = 0;
      if (mine && t0 + tb < t_hi) {
        const float2 v = *reinterpret_cast<const float2*>(
            a.hsave + ((b * nblk + (t0 + tb) / kSaveSteps) * a.Dm + d0 + ch) * NP + n0);
        h = pk(v.x, v.y);
      }
      {
        float py[RG], pc[2 * CG];
#pragma unroll
        for (int j = 0; j < kSaveSteps; ++j) {
          const float4 e = s_q[tb + j][ch];
          const f2 Bv = *reinterpret_cast<const f2*>(&s_b[tb + j][n0]);
          aa[j] = ex2_2(mul2(A2, pk(e.x, e.x)));
          ah[j] = mul2(aa[j], h);
          h = fma2(pk(e.y, e.y), Bv, ah[j]);
          if (zp_) {
            const float2 y = up(mul2(*reinterpret_cast<const f2*>(&s_c[tb + j][n0]), h));
            py[j % RG] = y.x + y.y;
            if (j % RG == RG - 1) put_row(py, tb + j + 1 - RG, s_y);
          }
          if (a.dbc) {
            const float2 c = up(mul2(pk(e.z, e.z), h));
            pc[j % CG * 2] = c.x, pc[j % CG * 2 + 1] = c.y;
            if (j % CG == CG - 1) put(pc, tb + j + 1 - CG, 1);
          }
        }
      }
      float p1[RG], p2[RG], pb[2 * CG];
#pragma unroll
      for (int j = kSaveSteps - 1; j >= 0; --j) {
        const float4 e = s_q[tb + j][ch];
        const f2 Bv = *reinterpret_cast<const f2*>(&s_b[tb + j][n0]);
        const f2 Cv = *reinterpret_cast<const f2*>(&s_c[tb + j][n0]);
        const f2 gg = fma2(Cv, pk(e.z, e.z), q);
        const f2 w = mul2(gg, ah[j]);
        const float2 x1 = up(mul2(gg, Bv)), x2 = up(mul2(w, A2));
        p1[j % RG] = x1.x + x1.y;
        p2[j % RG] = x2.x + x2.y;  // in units of A log2(e)
        dA = fma2(w, pk(e.x, e.x), dA);
        if (a.dbc) {
          const float2 c = up(mul2(gg, pk(e.y, e.y)));
          pb[j % CG * 2] = c.x, pb[j % CG * 2 + 1] = c.y;
          if (j % CG == 0) put(pb, tb + j, 0);
        }
        q = mul2(gg, aa[j]);
        if (j % RG == 0) {
          put_row(p1, tb + j, s_1);
          put_row(p2, tb + j, s_2);
        }
      }
    }
    __syncthreads();

    // the tile's rows: du, ddelta, dz; its share of d D and d bias
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int tt = rrow + v * RT::kRowStep;
      if (t0 + tt >= t_hi) continue;
      Vec<IO, W> o1, o2, o3;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float4 e = s_q[tt][rcol + i];
        const float uu = to_f(ru[v].v[i]), s1 = s_1[tt][rcol + i];
        float dx = fmaf(uu, s1, s_2[tt][rcol + i] * 0.6931471805599453f);
        if (a.softplus) dx *= sigmoid(to_f(rd[v].v[i]) + bias[i]);
        from_f(o1.v[i], fmaf(e.x, s1, Dv[i] * e.z));
        from_f(o2.v[i], dx);
        if (zp_) {
          const float zz = to_f(rz[v].v[i]), sg = sigmoid(zz), y = fmaf(Dv[i], uu, s_y[tt][rcol + i]);
          from_f(o3.v[i], to_f(ro[v].v[i]) * y * sg * fmaf(zz, 1.f - sg, 1.f));
        }
        accD[i] = fmaf(e.z, uu, accD[i]);
        accb[i] += dx;
      }
      const int64_t at = (b * a.T + t0 + tt) * a.Dm + d0;
      store_row<IO, W>((IO*)a.du + at, rcol, nc, a.vec, o1);
      store_row<IO, W>((IO*)a.ddelta + at, rcol, nc, a.vec, o2);
      if (zp_) store_row<IO, W>((IO*)a.dz + at, rcol, nc, a.vec, o3);
    }
    if (a.dbc) {
      const int64_t base = (((int64_t)gt * a.Bsz + b) * a.T + t0) * 2 * NP;
      for (int i = tid; i < kTT * 2 * NP; i += kBwdThr) {
        if (t0 + i / (2 * NP) >= t_hi) break;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += s_red[w * kTT * 2 * NP + i];
        a.dbc[base + i] = s;
      }
    }
  }

  const int64_t part = (int64_t)b * a.nchunk + chunk;
  if (mine) {
    *reinterpret_cast<float2*>(a.part_dA + (part * a.Dm + d0 + ch) * NP + n0) = up(dA);
    if (chunk == 0 && a.dh0) {
      const float2 v = up(q);
      float* o = a.dh0 + ((int64_t)b * a.Dm + d0 + ch) * a.N + n0;
      if (n0 < a.N) o[0] = v.x;
      if (n0 + 1 < a.N) o[1] = v.y;
    }
  }
  // d D, d bias over the threads that share a column
  float* red = reinterpret_cast<float*>(s_q);  // [2][kRowStep][CH]
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) {
    red[rrow * CH + rcol + i] = accD[i];
    red[(RT::kRowStep + rrow) * CH + rcol + i] = accb[i];
  }
  __syncthreads();
  if (tid < 2 * CH) {
    const int which = tid / CH, c = tid % CH;
    if (c < nc) {
      float s = 0.f;
      for (int r = 0; r < RT::kRowStep; ++r) s += red[(which * RT::kRowStep + r) * CH + c];
      a.part_dD[(part * 2 + which) * a.Dm + d0 + c] = s;
    }
  }
}

// d B, d C: the sum of the channel tiles' records, in tile order. One thread per 4 states; rows past the
// length hold zeros.
template <class IO, int NP>
__global__ void __launch_bounds__(256) k_sscan_dbc(const float* dbc, IO* dB, IO* dC, int64_t rows, int N, int G,
                                                   int tiles) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;  // over [rows, 2, NP] of group blockIdx.y
  if (i >= rows * 2 * NP) return;
  const int g = blockIdx.y;
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
