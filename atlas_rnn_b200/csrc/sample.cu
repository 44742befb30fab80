// C ABI of the token sampler (kernel in sample.cuh).
#include <atomic>

#include "launch.cuh"
#include "sample.cuh"

using namespace atlas;
using namespace atlas::smp;

namespace {

template <class IO, int NT>
constexpr int kBytes = (int)(sizeof(Smem) + sizeof(typename Row<IO, NT>::Ring));

template <class IO, int NT>
void configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& at, int64_t rows, int C, cudaStream_t st) {
  static_assert(kBytes<IO, NT> <= 227 * 1024, "shared memory");
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = C, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = kBytes<IO, NT>;
  cfg.stream = st;
  cfg.attrs = &at, cfg.numAttrs = C > 1;  // a plain launch for rows of one CTA
}

// Clusters of C CTAs that run at a time on the current device. Below 148 / C: a cluster stays within a group of SMs.
template <class IO, int NT>
int resident(int C) {
  static std::atomic<int> cached[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = cached[dev][C].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at = {};
    configure<IO, NT>(cfg, at, 1, C, nullptr);
    if (cudaOccupancyMaxActiveClusters(&n, k_sample<IO, NT>, &cfg) != cudaSuccess || n < 1) n = 1;
    cached[dev][C].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <class IO, int NT>
int launch(SampleArgs a, int64_t rows, cudaStream_t st) {
  if (cudaFuncSetAttribute(k_sample<IO, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes<IO, NT>) != cudaSuccess)
    return ATLAS_ERR_LAUNCH;
  // a row's CTAs: as many as still run in one wave (16 greedy rows of 131072: 6.6 us in clusters of 4, 9.7 in two
  // waves of clusters of 8), each with at least 4096 tokens
  int C = 8;
  while (C > 1 && (a.V / C < 4096 || rows > resident<IO, NT>(C))) C /= 2;
  a.split = (int)((((int64_t)a.V + C - 1) / C + 15) / 16 * 16);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at = {};
  configure<IO, NT>(cfg, at, rows, C, st);
  const int slot = prof_begin(KID_SAMPLE, st);
  if (cudaLaunchKernelEx(&cfg, k_sample<IO, NT>, a) != cudaSuccess) return ATLAS_ERR_LAUNCH;
  LAUNCH_CHECK();
  prof_end(slot, st);
  return ATLAS_OK;
}

}  // namespace

extern "C" int atlas_sample_tokens(const AtlasSample* p, void* stream) {
  if (!p || !p->logits || !p->noise || !p->out || p->rows < 1 || p->V < 1 || p->V > kMaxV ||
      (p->dtype != ATLAS_F32 && p->dtype != ATLAS_BF16) || p->rows > 0x7fffffff / 8)
    return ATLAS_ERR_INVALID_ARG;
  SampleArgs a = {};
  a.logits = p->logits, a.noise = p->noise, a.stride = p->stride, a.noise_stride = p->noise_stride, a.out = p->out;
  a.V = (int)p->V;
  a.temperature = p->temperature, a.top_p = p->top_p, a.min_p = p->min_p, a.top_k = p->top_k;
  a.temperature_row = p->temperature_row, a.top_p_row = p->top_p_row, a.min_p_row = p->min_p_row;
  a.top_k_row = p->top_k_row;
  cudaStream_t st = (cudaStream_t)stream;
  // long rows: 512 threads a CTA
  const bool wide = p->V > 4096;
  if (p->dtype == ATLAS_BF16)
    return wide ? launch<__nv_bfloat16, 512>(a, p->rows, st) : launch<__nv_bfloat16, 256>(a, p->rows, st);
  return wide ? launch<float, 512>(a, p->rows, st) : launch<float, 256>(a, p->rows, st);
}
