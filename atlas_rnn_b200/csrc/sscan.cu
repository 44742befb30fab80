// C ABI of the selective state space scan (kernels in sscan.cuh): argument checks, the
// plan of a call and its launches.
#include <algorithm>

#include "launch.cuh"
#include "sscan.cuh"

using namespace atlas;
using namespace atlas::ss;

namespace {

constexpr size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }

int mc_bwd(int np) { return np < 64 ? kMcBwd<8> : kMcBwd<64>; }
int padded(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

struct Plan {
  int np;             // padded state count
  int chunk, nchunk;  // time axis
};

constexpr int kMaxChunks = 65535;  // the second dimension of a grid

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

int tiles_of(const AtlasSelScan* a, int np, int mc) {  // channel tiles (CTAs) of one group
  const int ch = 32 / (np / kSpt) * mc * kWarps;
  return (a->D / a->G + ch - 1) / ch;
}

// Cut of the time axis of a pass whose CTAs cover mc channels a lane and fit `resident` times on an SM. One wave of
// CTAs where they fill the machine; the backward runs several smaller waves, whose tail weighs less against its longer
// chunks (B 4, T 8192, D 1536, N 16: 14% less in five waves than in one; the forward 5% more in two), as long
// as chunks keep 256 steps. None below 32 steps (T 512: 17 us for the forward, 25 with 64).
void cut(const AtlasSelScan* a, int mc, int resident, int waves, Plan& p) {
  p.np = padded(a->N);
  const int64_t ctas = a->B * a->G * tiles_of(a, p.np, mc), wave = (int64_t)sm_count() * resident;
  const int64_t fill = std::max<int64_t>(1, wave / ctas), many = std::max<int64_t>(1, waves * wave / ctas);
  auto steps = [&](int64_t n) { return (a->T + n - 1) / n; };
  int64_t c = std::max(steps(many), std::min<int64_t>(256, steps(fill)));
  if (waves > 1 && wave / ctas < 1) c = a->T;
  // a chunk asked for is lengthened where a grid could not hold as many of them
  const int64_t least = round_up((a->T + kMaxChunks - 1) / kMaxChunks, 32);
  c = a->chunk > 0 ? std::max<int64_t>(a->chunk, least) : round_up(std::max<int64_t>(c, 32), kTT);
  c = std::min<int64_t>(c, round_up(a->T, kTT));
  p.chunk = (int)std::min<int64_t>(c, (int64_t)1 << 30);
  p.nchunk = (int)((a->T + p.chunk - 1) / p.chunk);
}
Plan fwd_plan(const AtlasSelScan* a) {
  Plan p;
  cut(a, kMcFwd, kFwdCtas, 1, p);
  return p;
}
Plan bwd_plan(const AtlasSelScan* a) {
  Plan p;
  cut(a, mc_bwd(padded(a->N)), kBwdCtas, 5, p);
  return p;
}

bool sizes_ok(const AtlasSelScan* a) {
  return a && a->B >= 1 && a->T >= 1 && a->D >= 1 && a->N >= 1 && a->N <= 64 && a->G >= 1 && a->D % a->G == 0 &&
         (a->dtype_io == ATLAS_F32 || a->dtype_io == ATLAS_BF16) && a->chunk >= 0 && a->chunk % 32 == 0 &&
         a->B <= (1 << 24) && a->T <= 0x7fffffff && a->D <= (1 << 30) &&
         a->B * (int64_t)a->D * (a->N / 4 + 8) < ((int64_t)1 << 36);
}
bool inputs_ok(const AtlasSelScan* a) {
  return a->u && a->delta && a->Bm && a->Cm && a->A && (uintptr_t)a->saved % 16 == 0 && (uintptr_t)a->scratch % 16 == 0;
}

size_t saved_bytes(const AtlasSelScan* a) {
  return (size_t)a->B * ((a->T + kTT - 1) / kTT) * a->D * padded(a->N) * sizeof(float);
}
size_t ends_bytes(const AtlasSelScan* a, const Plan& p) {
  if (p.nchunk == 1) return 0;
  const size_t rows = (size_t)a->B * p.nchunk * a->D;
  return align_up(rows * p.np * sizeof(float)) + align_up(rows * sizeof(float));
}
struct BwdLayout {
  size_t dbc, dA, dD, ends, total;
};
BwdLayout bwd_layout(const AtlasSelScan* a, const Plan& p) {
  BwdLayout L;
  size_t at = 0;
  L.dbc = at;
  at += align_up((size_t)a->G * tiles_of(a, p.np, mc_bwd(p.np)) * a->B * a->T * 2 * p.np * sizeof(float));
  L.dA = at;
  at += align_up((size_t)a->B * p.nchunk * a->D * p.np * sizeof(float));
  L.dD = at;
  at += align_up((size_t)a->B * p.nchunk * 2 * a->D * sizeof(float));
  L.ends = at;
  L.total = at + ends_bytes(a, p);
  return L;
}

ScanArgs pack(const AtlasSelScan* a, const Plan& p) {
  ScanArgs s = {};
  s.u = a->u, s.delta = a->delta, s.z = a->z, s.Bm = a->Bm, s.Cm = a->Cm, s.dout = a->dout;
  s.u_sb = a->u_sb, s.u_st = a->u_st, s.d_sb = a->delta_sb, s.d_st = a->delta_st, s.z_sb = a->z_sb, s.z_st = a->z_st;
  s.o_sb = a->dout_sb, s.o_st = a->dout_st;
  s.B_sb = a->B_sb, s.B_st = a->B_st, s.B_sg = a->B_sg, s.C_sb = a->C_sb, s.C_st = a->C_st, s.C_sg = a->C_sg;
  s.A = a->A, s.D = a->Dskip, s.bias = a->bias, s.h0 = a->h0, s.len = a->len;
  s.out = a->out, s.hT = a->hT;
  s.dhT = a->dhT, s.du = a->du, s.ddelta = a->ddelta, s.dz = a->dz, s.dh0 = a->dh0;
  s.T = a->T, s.Bsz = (int)a->B, s.Dm = a->D, s.N = a->N, s.G = a->G, s.softplus = a->softplus;
  s.chunk = p.chunk, s.nchunk = p.nchunk;
  return s;
}

// Whether rows of `p` allow accesses of W neighbouring elements at multiples of W.
bool wide(const void* p, int64_t sb, int64_t st, int size, int W) {
  return !p || ((uintptr_t)p % (size_t)(W * size) == 0 && sb % W == 0 && st % W == 0);
}
// vec, vecbc: 16-byte pieces of the rows read, of B and C (one token: 4 elements of them); pair: two elements of the rows written.
void alignment(const AtlasSelScan* a, ScanArgs& s, int bc) {
  const int size = a->dtype_io == ATLAS_BF16 ? 2 : 4, E = 16 / size;
  const int64_t dg = a->G == 1 ? 0 : a->D / a->G;
  s.vec = wide(a->u, a->u_sb, a->u_st, size, E) && wide(a->delta, a->delta_sb, a->delta_st, size, E) &&
          wide(a->z, a->z_sb, a->z_st, size, E) && wide(a->dout, a->dout_sb, a->dout_st, size, E) && dg % E == 0;
  s.pair = wide(a->out, a->D, a->D, size, 2) && wide(a->du, a->D, a->D, size, 2) &&
           wide(a->ddelta, a->D, a->D, size, 2) && wide(a->dz, a->D, a->D, size, 2) && dg % 2 == 0;
  s.vecbc = wide(a->Bm, a->B_sb, a->B_st, size, bc) && wide(a->Cm, a->C_sb, a->C_st, size, bc) &&
            (a->G == 1 || (a->B_sg % bc == 0 && a->C_sg % bc == 0));
}

// A walking kernel over (batch x groups x channel tiles, chunks) with its warps' shared memory.
template <class K>
int walk(int kid, K kernel, const AtlasSelScan* a, const ScanArgs& s, int tiles, int chunks, int bytes, cudaStream_t st) {
  const int64_t gx = a->B * a->G * tiles;
  if (gx > 0x7fffffff || chunks > kMaxChunks) return ATLAS_ERR_UNSUPPORTED;
  if (bytes > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return ATLAS_ERR_LAUNCH;
  LAUNCH_T(kid, kernel, dim3((unsigned)gx, chunks), 32 * kWarps, bytes, st, s);
  return ATLAS_OK;
}

template <int NP, bool BACK>
int carry(const AtlasSelScan* a, const ScanArgs& s, cudaStream_t st) {
  const int64_t n = a->B * a->D * (NP / 4), grid = (n + kCarryThr - 1) / kCarryThr;
  if (grid > 0x7fffffff) return ATLAS_ERR_UNSUPPORTED;
  LAUNCH_T(KID_SSCAN_CARRY, (k_sscan_carry<NP, BACK>), dim3((unsigned)grid), kCarryThr, 0, st, s);
  return ATLAS_OK;
}

template <class IO, int NP, bool Z>
int fwd_t(const AtlasSelScan* a, ScanArgs s, cudaStream_t st) {
  const int tiles = tiles_of(a, NP, kMcFwd);
  alignment(a, s, 16 / (int)sizeof(IO));
  if (s.nchunk > 1) {
    if (const int rc = walk(KID_SSCAN_ENDS, k_sscan_fwd<IO, NP, true, false>, a, s, tiles, s.nchunk - 1,
                            kWarps * (int)sizeof(FwdSmem<IO, NP, true, false>), st))
      return rc;
    if (const int rc = carry<NP, false>(a, s, st)) return rc;
  }
  return walk(KID_SSCAN_FWD, k_sscan_fwd<IO, NP, false, Z>, a, s, tiles, s.nchunk,
              kWarps * (int)sizeof(FwdSmem<IO, NP, false, Z>), st);
}

template <class IO, int NP>
int step_t(const AtlasSelScan* a, ScanArgs s, cudaStream_t st) {
  alignment(a, s, 4);
  const bool v4 = s.vecbc && a->N % 4 == 0 && (uintptr_t)a->A % 16 == 0 && (uintptr_t)a->h0 % 16 == 0 &&
                   (uintptr_t)a->hT % 16 == 0;
  // four rows a thread where one row each would give an SM eight CTAs (D 1536, N 16, bf16: 16 rows 2.2 us with one, 2.4 with
  // four; 32 rows 3.8 and 3.6; 128 rows 8.8 and 6.7)
  const int64_t per = kStepThr / (NP / 4), gx = (a->D + per - 1) / per, rows = a->B * gx >= 8 * 148 ? 4 : 1;
  const int64_t gy = (a->B + rows - 1) / rows;
  if (gx > 0x7fffffff || gy > 65535) return ATLAS_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (rows == 4 && v4) LAUNCH_T(KID_SSCAN_STEP, (k_sscan_step<IO, NP, 4, true>), grid, kStepThr, 0, st, s);
  else if (rows == 4) LAUNCH_T(KID_SSCAN_STEP, (k_sscan_step<IO, NP, 4, false>), grid, kStepThr, 0, st, s);
  else if (v4) LAUNCH_T(KID_SSCAN_STEP, (k_sscan_step<IO, NP, 1, true>), grid, kStepThr, 0, st, s);
  else LAUNCH_T(KID_SSCAN_STEP, (k_sscan_step<IO, NP, 1, false>), grid, kStepThr, 0, st, s);
  return ATLAS_OK;
}

template <class IO, int NP, bool Z>
int bwd_t(const AtlasSelScan* a, ScanArgs s, const BwdLayout& L, cudaStream_t st) {
  const int64_t rows = a->B * a->T, blocks = (rows * 2 * NP / 4 + 255) / 256;
  if (a->dB && blocks > 0x7fffffff / a->G) return ATLAS_ERR_UNSUPPORTED;  // before the first launch
  const int tiles = tiles_of(a, NP, kMcBwd<NP>);
  alignment(a, s, 16 / (int)sizeof(IO));
  if (s.nchunk > 1) {
    if (const int rc = walk(KID_SSCAN_BWD_ENDS, k_sscan_bwd_ends<IO, NP, Z>, a, s, tiles, s.nchunk - 1,
                            kWarps * (int)sizeof(EndsSmem<IO, NP, Z>), st))
      return rc;
    if (const int rc = carry<NP, true>(a, s, st)) return rc;
  }
  if (const int rc = walk(KID_SSCAN_BWD, k_sscan_bwd<IO, NP, Z>, a, s, tiles, s.nchunk, (int)sizeof(BwdSmem<IO, NP, Z>), st))
    return rc;
  if (a->dB) {
    LAUNCH_T(KID_SSCAN_DBC, (k_sscan_dbc<IO, NP>), dim3((unsigned)(blocks * a->G)), 256, 0, st, s.dbc, (IO*)a->dB,
             (IO*)a->dC, rows, a->N, a->G, tiles_of(a, NP, kMcBwd<NP>), (unsigned)blocks);
  }
  const int64_t n = (int64_t)a->D * NP + 2 * (int64_t)a->D;
  LAUNCH_T(KID_SSCAN_DA, k_sscan_dA, dim3((unsigned)((n + 255) / 256)), 256, 0, st, s.part_dA, s.part_dD, a->dA, a->dD,
           a->dbias, (int)(a->B * s.nchunk), a->D, a->N, NP);
  return ATLAS_OK;
}

template <class IO>
int fwd_io(const AtlasSelScan* a, const Plan& p, const ScanArgs& s, cudaStream_t st) {
  if (a->T == 1 && !s.hsave && a->B <= 65535) {
    switch (p.np) {
      case 8: return step_t<IO, 8>(a, s, st);
      case 16: return step_t<IO, 16>(a, s, st);
      case 32: return step_t<IO, 32>(a, s, st);
      default: return step_t<IO, 64>(a, s, st);
    }
  }
  switch (p.np) {
    case 8: return a->z ? fwd_t<IO, 8, true>(a, s, st) : fwd_t<IO, 8, false>(a, s, st);
    case 16: return a->z ? fwd_t<IO, 16, true>(a, s, st) : fwd_t<IO, 16, false>(a, s, st);
    case 32: return a->z ? fwd_t<IO, 32, true>(a, s, st) : fwd_t<IO, 32, false>(a, s, st);
    default: return a->z ? fwd_t<IO, 64, true>(a, s, st) : fwd_t<IO, 64, false>(a, s, st);
  }
}
template <class IO>
int bwd_io(const AtlasSelScan* a, const Plan& p, const ScanArgs& s, const BwdLayout& L, cudaStream_t st) {
  switch (p.np) {
    case 8: return a->z ? bwd_t<IO, 8, true>(a, s, L, st) : bwd_t<IO, 8, false>(a, s, L, st);
    case 16: return a->z ? bwd_t<IO, 16, true>(a, s, L, st) : bwd_t<IO, 16, false>(a, s, L, st);
    case 32: return a->z ? bwd_t<IO, 32, true>(a, s, L, st) : bwd_t<IO, 32, false>(a, s, L, st);
    default: return a->z ? bwd_t<IO, 64, true>(a, s, L, st) : bwd_t<IO, 64, false>(a, s, L, st);
  }
}

}  // namespace

extern "C" {

int atlas_sscan_workspace(const AtlasSelScan* a, size_t* saved, size_t* fwd_scratch, size_t* bwd_scratch) {
  if (!sizes_ok(a) || !saved || !fwd_scratch || !bwd_scratch) return ATLAS_ERR_INVALID_ARG;
  *saved = saved_bytes(a);
  *fwd_scratch = ends_bytes(a, fwd_plan(a));
  *bwd_scratch = bwd_layout(a, bwd_plan(a)).total;
  return ATLAS_OK;
}

int atlas_sscan_forward(const AtlasSelScan* a, void* stream) {
  if (!sizes_ok(a) || !inputs_ok(a) || !a->out || !a->hT) return ATLAS_ERR_INVALID_ARG;
  const Plan p = fwd_plan(a);
  const size_t ends = ends_bytes(a, p);
  if ((a->saved && a->saved_bytes < saved_bytes(a)) || (ends && (!a->scratch || a->scratch_bytes < ends)))
    return ATLAS_ERR_WORKSPACE;
  ScanArgs s = pack(a, p);
  s.hsave = (float*)a->saved;
  if (ends) {
    s.part_h = (float*)a->scratch;
    s.part_dt = (float*)((char*)a->scratch + align_up((size_t)a->B * p.nchunk * a->D * p.np * sizeof(float)));
  }
  cudaStream_t st = (cudaStream_t)stream;
  return a->dtype_io == ATLAS_BF16 ? fwd_io<__nv_bfloat16>(a, p, s, st) : fwd_io<float>(a, p, s, st);
}

int atlas_sscan_backward(const AtlasSelScan* a, void* stream) {
  if (!sizes_ok(a) || !inputs_ok(a) || !a->dout || !a->du || !a->ddelta || !a->dA || (a->z && !a->dz) ||
      !a->dB != !a->dC)
    return ATLAS_ERR_INVALID_ARG;
  const Plan p = bwd_plan(a);
  const BwdLayout L = bwd_layout(a, p);
  if (!a->saved || a->saved_bytes < saved_bytes(a) || !a->scratch || a->scratch_bytes < L.total)
    return ATLAS_ERR_WORKSPACE;
  ScanArgs s = pack(a, p);
  char* w = (char*)a->scratch;
  s.hsave = (float*)a->saved;
  s.dbc = (float*)(w + L.dbc);
  s.part_dA = (float*)(w + L.dA);
  s.part_dD = (float*)(w + L.dD);
  if (p.nchunk > 1) {
    s.part_h = (float*)(w + L.ends);
    s.part_dt = (float*)(w + L.ends + align_up((size_t)a->B * p.nchunk * a->D * p.np * sizeof(float)));
  }
  cudaStream_t st = (cudaStream_t)stream;
  return a->dtype_io == ATLAS_BF16 ? bwd_io<__nv_bfloat16>(a, p, s, L, st) : bwd_io<float>(a, p, s, L, st);
}

}  // extern "C"
