// C ABI of the selective state space scan (kernels in sscan.cuh): argument checks, the
// plan of a call and its launches.
#include <algorithm>

#include "launch.cuh"
#include "sscan.cuh"

using namespace atlas;
using namespace atlas::ss;

namespace {

constexpr size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }

int padded(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

struct Plan {
  int np, spt;        // padded state count, states per lane (forward)
  int chunk, nchunk;  // time axis
};

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Cut of the time axis: none while the rows and channels fill the machine, else enough chunks for it.
void cut(const AtlasSelScan* a, int64_t warps, int64_t want, Plan& p) {
  int64_t n = warps >= want ? 1 : std::min<int64_t>((want + warps - 1) / warps, 16);
  int64_t c = a->chunk > 0 ? a->chunk : round_up((a->T + n - 1) / n, kTT);
  if (c < 8 * kTT && a->chunk <= 0) c = 8 * kTT;
  c = std::min<int64_t>(c, round_up(a->T, kTT));
  p.chunk = (int)std::min<int64_t>(c, (int64_t)1 << 30);
  p.nchunk = (int)((a->T + p.chunk - 1) / p.chunk);
}

Plan fwd_plan(const AtlasSelScan* a) {
  Plan p;
  p.np = padded(a->N);
  const int64_t sms = 148;
  const int64_t w4 = (int64_t)a->B * a->D * (p.np / 4) / 32;
  p.spt = w4 >= sms * 8 ? 4 : 2;
  int64_t want = sms * 6;
  cut(a, std::max<int64_t>(1, p.spt == 4 ? w4 : 2 * w4), want, p);
  return p;
}
Plan bwd_plan(const AtlasSelScan* a) {
  Plan p;
  p.np = padded(a->N);
  p.spt = 2;
  const int64_t w = std::max<int64_t>(1, (int64_t)a->B * a->D * (p.np / 2) / 32);
  int64_t want = 148 * 8;
  cut(a, w, want, p);
  return p;
}

bool sizes_ok(const AtlasSelScan* a) {
  return a && a->B >= 1 && a->T >= 1 && a->D >= 1 && a->N >= 1 && a->N <= 64 && a->G >= 1 && a->D % a->G == 0 &&
         (a->dtype_io == ATLAS_F32 || a->dtype_io == ATLAS_BF16) && a->chunk >= 0 && a->chunk % kTT == 0 &&
         a->B <= (1 << 24) && a->T <= ((int64_t)1 << 40) &&
         a->B * (int64_t)a->D * (a->N / 4 + 8) < ((int64_t)1 << 36);
}
bool inputs_ok(const AtlasSelScan* a) { return a->u && a->delta && a->Bm && a->Cm && a->A; }

size_t saved_bytes(const AtlasSelScan* a) {
  return (size_t)a->B * ((a->T + kSaveSteps - 1) / kSaveSteps) * a->D * padded(a->N) * sizeof(float);
}
size_t ends_bytes(const AtlasSelScan* a, const Plan& p) {
  if (p.nchunk == 1) return 0;
  const size_t rows = (size_t)a->B * p.nchunk * a->D;
  return align_up(rows * p.np * sizeof(float)) + align_up(rows * sizeof(float));
}
int bwd_tiles(const AtlasSelScan* a, int np) {  // channel tiles of one group
  const int ch = kBwdThr / (np / 2);
  return (a->D / a->G + ch - 1) / ch;
}
struct BwdLayout {
  size_t dbc, dA, dD, ends, total;
};
BwdLayout bwd_layout(const AtlasSelScan* a, const Plan& p) {
  BwdLayout L;
  size_t at = 0;
  L.dbc = at;
  at += align_up((size_t)a->G * bwd_tiles(a, p.np) * a->B * a->T * 2 * p.np * sizeof(float));
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
void alignment(const AtlasSelScan* a, ScanArgs& s, int W, bool bwd) {
  const int size = a->dtype_io == ATLAS_BF16 ? 2 : 4;
  s.vec = wide(a->u, a->u_sb, a->u_st, size, W) && wide(a->delta, a->delta_sb, a->delta_st, size, W) &&
          wide(a->z, a->z_sb, a->z_st, size, W) && wide(a->out, a->D, a->D, size, W) &&
          (a->G == 1 || a->D / a->G % W == 0);
  if (bwd)
    s.vec = s.vec && wide(a->dout, a->dout_sb, a->dout_st, size, W) && wide(a->du, a->D, a->D, size, W) &&
            wide(a->ddelta, a->D, a->D, size, W) && wide(a->dz, a->D, a->D, size, W);
  s.vecbc = wide(a->Bm, a->B_sb, a->B_st, size, 4) && wide(a->Cm, a->C_sb, a->C_st, size, 4) &&
            (a->G == 1 || (a->B_sg % 4 == 0 && a->C_sg % 4 == 0));
}

template <class IO, int NP, int SPT>
int fwd_t(const AtlasSelScan* a, ScanArgs s, cudaStream_t st) {
  constexpr int CH = kFwdThr / (NP / SPT);
  alignment(a, s, RowTile<IO, CH, kFwdThr, kTT>::W, false);
  const int64_t gx = a->B * a->G * ((a->D / a->G + CH - 1) / CH);
  if (gx > 0x7fffffff || s.nchunk > 65535) return ATLAS_ERR_UNSUPPORTED;
  if (s.nchunk > 1)
    LAUNCH_T(KID_SSCAN_ENDS, (k_sscan_fwd<IO, NP, SPT, true>), dim3((unsigned)gx, s.nchunk - 1), kFwdThr, 0, st, s);
  LAUNCH_T(KID_SSCAN_FWD, (k_sscan_fwd<IO, NP, SPT, false>), dim3((unsigned)gx, s.nchunk), kFwdThr, 0, st, s);
  return ATLAS_OK;
}

template <class IO, int NP>
int step_t(const AtlasSelScan* a, ScanArgs s, cudaStream_t st) {
  alignment(a, s, 1, false);
  const int vec4 = a->N % 4 == 0 && (uintptr_t)a->A % 16 == 0 && (uintptr_t)a->h0 % 16 == 0 &&
                   (uintptr_t)a->hT % 16 == 0;
  const int64_t per = kStepThr / (NP / 4), grid = (a->B * a->D + per - 1) / per;
  if (grid > 0x7fffffff) return ATLAS_ERR_UNSUPPORTED;
  LAUNCH_T(KID_SSCAN_STEP, (k_sscan_step<IO, NP>), dim3((unsigned)grid), kStepThr, 0, st, s, vec4);
  return ATLAS_OK;
}

template <class IO, int NP>
int bwd_t(const AtlasSelScan* a, ScanArgs s, const BwdLayout& L, cudaStream_t st) {
  constexpr int CH = BwdSmem<NP>::CH, FCH = kFwdThr / (NP / 2);
  const int64_t dg = a->D / a->G, tiles = (dg + CH - 1) / CH, gx = a->B * a->G * tiles;
  const int64_t rows = a->B * a->T;
  if (gx > 0x7fffffff || s.nchunk > 65535) return ATLAS_ERR_UNSUPPORTED;
  if (s.nchunk > 1) {
    ScanArgs e = s;
    alignment(a, e, RowTile<IO, FCH, kFwdThr, kTT>::W, true);
    const int64_t ex = a->B * a->G * ((dg + FCH - 1) / FCH);
    if (ex > 0x7fffffff) return ATLAS_ERR_UNSUPPORTED;
    LAUNCH_T(KID_SSCAN_BWD_ENDS, (k_sscan_bwd_ends<IO, NP, 2>), dim3((unsigned)ex, s.nchunk - 1), kFwdThr, 0, st, e);
  }
  alignment(a, s, RowTile<IO, CH, kBwdThr, kTT>::W, true);
  if (cudaFuncSetAttribute(k_sscan_bwd<IO, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<NP>::bytes) !=
      cudaSuccess)
    return ATLAS_ERR_LAUNCH;
  LAUNCH_T(KID_SSCAN_BWD, (k_sscan_bwd<IO, NP>), dim3((unsigned)gx, s.nchunk), kBwdThr, BwdSmem<NP>::bytes, st, s);
  if (s.dbc) {
    const int64_t blocks = (rows * 2 * NP / 4 + 255) / 256;
    if (blocks > 0x7fffffff || a->G > 65535) return ATLAS_ERR_UNSUPPORTED;
    LAUNCH_T(KID_SSCAN_DBC, (k_sscan_dbc<IO, NP>), dim3((unsigned)blocks, a->G), 256, 0, st, s.dbc, (IO*)a->dB,
             (IO*)a->dC, rows, a->N, a->G, (int)tiles);
  }
  const int64_t n = (int64_t)a->D * NP + 2 * (int64_t)a->D;
  LAUNCH_T(KID_SSCAN_DA, k_sscan_dA, dim3((unsigned)((n + 255) / 256)), 256, 0, st, s.part_dA, s.part_dD, a->dA, a->dD,
           a->dbias, (int)(a->B * s.nchunk), a->D, a->N, NP);
  return ATLAS_OK;
}

template <class IO>
int fwd_io(const AtlasSelScan* a, const Plan& p, const ScanArgs& s, cudaStream_t st) {
  if (a->T == 1 && !s.hsave) {
    switch (p.np) {
      case 8: return step_t<IO, 8>(a, s, st);
      case 16: return step_t<IO, 16>(a, s, st);
      case 32: return step_t<IO, 32>(a, s, st);
      default: return step_t<IO, 64>(a, s, st);
    }
  }
  switch (p.np * 10 + p.spt) {
    case 82: return fwd_t<IO, 8, 2>(a, s, st);
    case 84: return fwd_t<IO, 8, 4>(a, s, st);
    case 162: return fwd_t<IO, 16, 2>(a, s, st);
    case 164: return fwd_t<IO, 16, 4>(a, s, st);
    case 322: return fwd_t<IO, 32, 2>(a, s, st);
    case 324: return fwd_t<IO, 32, 4>(a, s, st);
    case 642: return fwd_t<IO, 64, 2>(a, s, st);
    default: return fwd_t<IO, 64, 4>(a, s, st);
  }
}
template <class IO>
int bwd_io(const AtlasSelScan* a, const Plan& p, const ScanArgs& s, const BwdLayout& L, cudaStream_t st) {
  switch (p.np) {
    case 8: return bwd_t<IO, 8>(a, s, L, st);
    case 16: return bwd_t<IO, 16>(a, s, L, st);
    case 32: return bwd_t<IO, 32>(a, s, L, st);
    default: return bwd_t<IO, 64>(a, s, L, st);
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
  s.dbc = a->dB ? (float*)(w + L.dbc) : nullptr;
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
