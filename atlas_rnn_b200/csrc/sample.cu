// C ABI of the token sampler (kernel in sample.cuh).
#include <algorithm>

#include "launch.cuh"
#include "sample.cuh"

using namespace atlas;
using namespace atlas::smp;

namespace {

template <class IO, int NT>
int launch(const SampleArgs& a, int64_t rows, int C, cudaStream_t st) {
  static_assert(sizeof(Smem) <= 100 * 1024, "shared memory");
  if (cudaFuncSetAttribute(k_sample<IO, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem)) != cudaSuccess)
    return ATLAS_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = C, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = sizeof(Smem);
  cfg.stream = st;
  cfg.attrs = &at, cfg.numAttrs = 1;
  const int slot = prof_begin(KID_SAMPLE, st);
  if (cudaLaunchKernelEx(&cfg, k_sample<IO, NT>, a) != cudaSuccess) return ATLAS_ERR_LAUNCH;
  LAUNCH_CHECK();
  prof_end(slot, st);
  return ATLAS_OK;
}

}  // namespace

extern "C" int atlas_sample_tokens(const AtlasSample* p, void* stream) {
  if (!p || !p->logits || !p->noise || !p->out || p->rows < 1 || p->V < 1 || p->V > 0x7ffffff0 ||
      (p->dtype != ATLAS_F32 && p->dtype != ATLAS_BF16) || p->rows > 0x7fffffff / 8)
    return ATLAS_ERR_INVALID_ARG;
  SampleArgs a = {};
  a.logits = p->logits, a.noise = p->noise, a.stride = p->stride, a.noise_stride = p->noise_stride, a.out = p->out;
  a.V = (int)p->V;
  a.temperature = p->temperature, a.top_p = p->top_p, a.min_p = p->min_p, a.top_k = p->top_k;
  a.temperature_row = p->temperature_row, a.top_p_row = p->top_p_row, a.min_p_row = p->min_p_row;
  a.top_k_row = p->top_k_row;
  // a row's CTAs: as many as leave the machine one CTA an SM, each with at least 4096 tokens
  int C = 8;
  while (C > 1 && (p->rows * C > sm_count() || p->V / C < 4096)) C /= 2;
  const int64_t split = ((p->V + C - 1) / C + 15) / 16 * 16;
  a.split = (int)split;
  const int size = p->dtype == ATLAS_BF16 ? 2 : 4, E = 16 / size;
  a.vec = (uintptr_t)p->logits % 16 == 0 && p->stride % E == 0;
  cudaStream_t st = (cudaStream_t)stream;
  const bool wide = split > 4096;
  if (p->dtype == ATLAS_BF16)
    return wide ? launch<__nv_bfloat16, 1024>(a, p->rows, C, st) : launch<__nv_bfloat16, 256>(a, p->rows, C, st);
  return wide ? launch<float, 1024>(a, p->rows, C, st) : launch<float, 256>(a, p->rows, C, st);
}
