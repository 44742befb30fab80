// C ABI of the distillation loss over a teacher's top logits (kernels in distill.cuh).
#include <algorithm>

#include "launch.cuh"
#include "distill.cuh"

using namespace atlas;
using namespace atlas::dst;

// 128 threads a CTA: the end of a row is a chain of small steps, which many rows an SM hide (8192 x 32000, bf16, forward:
// 103 us; 256 threads took 1.27 times as long, 64 1.36 times).
constexpr int kThr = 128;

namespace {

bool pack(const AtlasDistill* p, DistillArgs& a, int& C) {
  if (!p || !p->logits || !p->values || !p->indices || !p->stats || p->rows < 1 || p->V < 1 || p->V > 0x7ffffff0 ||
      p->K < 1 || p->K > kMaxK || (p->dtype != ATLAS_F32 && p->dtype != ATLAS_BF16) || !(p->temperature >= 0.99e-6f && p->temperature <= 1.01e6f) ||
      p->rows > 0x7fffffff / 8 || (uintptr_t)p->stats % 16)
    return false;
  a.logits = p->logits, a.stride = p->stride, a.values = p->values, a.indices = p->indices;
  a.loss = p->loss, a.valid = p->valid, a.stats = p->stats, a.dloss = p->dloss, a.dlogits = p->dlogits;
  a.V = (int)p->V, a.K = (int)p->K, a.rows = (int)p->rows, a.tau = p->temperature;
  // a row's CTAs: one where the rows fill the machine, else up to 8 with at least 4096 tokens each
  C = 8;
  while (C > 1 && (p->rows * C > 4 * sm_count() || p->V / C < 4096)) C /= 2;
  a.split = (int)(((p->V + C - 1) / C + 15) / 16 * 16);
  return true;
}

bool short_rows(const DistillArgs& a) { return a.V <= kShortV && a.K <= kShortK; }

template <class IO, int NT>
int fwd(const DistillArgs& a, int64_t rows, int C, cudaStream_t st) {
  if (short_rows(a)) {
    LAUNCH_T(KID_DISTILL_FWD, (k_distill_fwd<IO, 32, kShortRows>), dim3((unsigned)((rows + kShortRows - 1) / kShortRows)),
             32 * kShortRows, 0, st, a);
    return ATLAS_OK;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = C, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cfg.attrs = &at, cfg.numAttrs = C > 1;  // plain launches where they do: CTAs start faster (8192 x 32000: 103 us, not 115)
  const int slot = prof_begin(KID_DISTILL_FWD, st);
  if (cudaLaunchKernelEx(&cfg, k_distill_fwd<IO, NT, 1>, a) != cudaSuccess) return ATLAS_ERR_LAUNCH;
  LAUNCH_CHECK();
  prof_end(slot, st);
  return ATLAS_OK;
}
template <class IO, int NT>
int bwd(const DistillArgs& a, int64_t rows, int C, cudaStream_t st) {
  if (short_rows(a)) {
    LAUNCH_T(KID_DISTILL_BWD, (k_distill_bwd<IO, 32, kShortRows>), dim3((unsigned)((rows + kShortRows - 1) / kShortRows)),
             32 * kShortRows, 0, st, a, 1);
    return ATLAS_OK;
  }
  LAUNCH_T(KID_DISTILL_BWD, (k_distill_bwd<IO, NT, 1>), dim3((unsigned)(rows * C)), NT, 0, st, a, C);
  return ATLAS_OK;
}

}  // namespace

extern "C" {

int atlas_distill_forward(const AtlasDistill* p, void* stream) {
  DistillArgs a = {};
  int C;
  if (!pack(p, a, C) || !p->loss || !p->valid) return ATLAS_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  return p->dtype == ATLAS_BF16 ? fwd<__nv_bfloat16, kThr>(a, p->rows, C, st) : fwd<float, kThr>(a, p->rows, C, st);
}

int atlas_distill_backward(const AtlasDistill* p, void* stream) {
  DistillArgs a = {};
  int C;
  if (!pack(p, a, C) || !p->dloss || !p->dlogits) return ATLAS_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  return p->dtype == ATLAS_BF16 ? bwd<__nv_bfloat16, kThr>(a, p->rows, C, st) : bwd<float, kThr>(a, p->rows, C, st);
}

}  // extern "C"
