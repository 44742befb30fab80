// C ABI of the causal depthwise convolution (kernels in causal_conv.cuh).
#include <algorithm>

#include "launch.cuh"
#include "causal_conv.cuh"

using namespace atlas;
using namespace atlas::cc;

namespace {

// Steps per thread; shorter while the machine would not be filled. Forward 64. Backward 256: a run starts and ends with
// steps one by one (B 4, T 8192, C 1536, bf16: 125 us with 64, 110 with 128, 101 with 256).
int run_of(int64_t B, int64_t T, int64_t C, bool bwd) {
  int run = bwd ? 256 : 64;
  const int64_t want = 148 * (bwd ? 256 : 1024);
  while (run > 8 && B * ((T + run - 1) / run) * ((C + 3) / 4) < want) run /= 2;
  return run;
}
int ygrid_of(int64_t T, int run) { return (int)((T + (int64_t)run * kConvWarps - 1) / ((int64_t)run * kConvWarps)); }

bool shape_ok(int K, int dtype, int64_t B, int64_t T, int64_t C) {
  return K >= 2 && K <= 8 && (dtype == ATLAS_F32 || dtype == ATLAS_BF16) && B >= 1 && T >= 1 && C >= 1 &&
         C <= ((int64_t)1 << 20) && T <= 0x7fffffff &&
         B <= 0x7fffffff / std::max(1, ygrid_of(T, 8));
}
bool wide(const void* p, int64_t sb, int64_t st, int size, int W) {
  return !p || ((uintptr_t)p % (size_t)(W * size) == 0 && sb % W == 0 && st % W == 0);
}

template <int K, class IO, int W>
int launch(bool fwd, ConvArgs a, int64_t B, float* dw, float* dbias, cudaStream_t st) {
  const int size = (int)sizeof(IO);
  a.vec = wide(a.x, a.x_sb, a.x_st, size, W) && wide(a.init, a.C, a.C, size, W) && wide(a.dy, a.dy_sb, a.dy_st, size, W) &&
          wide(a.d_final, a.C, a.C, size, W) && wide(a.y, a.C, a.C, size, W) && wide(a.final_state, a.C, a.C, size, W) &&
          wide(a.dx, a.C, a.C, size, W) && wide(a.d_init, a.C, a.C, size, W);
  const dim3 grid((unsigned)(B * a.ygrid), (unsigned)((a.C + 32 * W - 1) / (32 * W)));
  if (fwd && a.T == 1 && B <= 65535) {
    // four rows a thread where one row each would give an SM two CTAs (C 1536, K 4, bf16: 64 rows 2.2 us with one, 2.4 with
    // four; 128 rows 2.8 and 2.5; 4096 rows 28.9 and 18.9)
    const int64_t gx = (a.C + kConvStepThr * W - 1) / (kConvStepThr * W), R = gx * B >= 2 * 148 ? 4 : 1;
    const dim3 one((unsigned)gx, (unsigned)((B + R - 1) / R));
    const bool fast = a.vec && a.C % W == 0 && (uintptr_t)a.w % 16 == 0;
    a.rows = B;
    if (fast && R == 4) LAUNCH_T(KID_CONV_STEP, (k_causal_conv_step<K, IO, W, 4, true>), one, kConvStepThr, 0, st, a);
    else if (fast) LAUNCH_T(KID_CONV_STEP, (k_causal_conv_step<K, IO, W, 1, true>), one, kConvStepThr, 0, st, a);
    else if (R == 4) LAUNCH_T(KID_CONV_STEP, (k_causal_conv_step<K, IO, W, 4, false>), one, kConvStepThr, 0, st, a);
    else LAUNCH_T(KID_CONV_STEP, (k_causal_conv_step<K, IO, W, 1, false>), one, kConvStepThr, 0, st, a);
    return ATLAS_OK;
  }
  if (fwd) {
    LAUNCH_T(KID_CONV_FWD, (k_causal_conv_fwd<K, IO, W>), grid, 32 * kConvWarps, 0, st, a);
    return ATLAS_OK;
  }
  LAUNCH_T(KID_CONV_BWD, (k_causal_conv_bwd<K, IO, W>), grid, 32 * kConvWarps, 0, st, a);
  const int64_t n = a.C * (K + 1);
  LAUNCH_T(KID_CONV_DW, k_causal_conv_dw, dim3((unsigned)((n + 31) / 32)), 256, 0, st, a.part, dw, dbias, n, K,
           B * a.ygrid);
  return ATLAS_OK;
}

// 4 channels a thread; 2 where more than 4 taps would take too many registers.
template <class IO>
int dispatch(bool fwd, int K, const ConvArgs& a, int64_t B, float* dw, float* dbias, cudaStream_t st) {
  switch (K) {
    case 2: return launch<2, IO, 4>(fwd, a, B, dw, dbias, st);
    case 3: return launch<3, IO, 4>(fwd, a, B, dw, dbias, st);
    case 4: return launch<4, IO, 4>(fwd, a, B, dw, dbias, st);
    case 5: return launch<5, IO, 2>(fwd, a, B, dw, dbias, st);
    case 6: return launch<6, IO, 2>(fwd, a, B, dw, dbias, st);
    case 7: return launch<7, IO, 2>(fwd, a, B, dw, dbias, st);
    default: return launch<8, IO, 2>(fwd, a, B, dw, dbias, st);
  }
}

}  // namespace

extern "C" {

int atlas_causal_conv_forward(const void* x, int64_t x_sb, int64_t x_st, const float* w, const float* bias,
                              const void* init, const int32_t* len, void* y, void* final_state, int K, int silu,
                              int dtype_io, int64_t B, int64_t T, int64_t C, void* stream) {
  if (!x || !w || !y || !final_state || !shape_ok(K, dtype_io, B, T, C)) return ATLAS_ERR_INVALID_ARG;
  ConvArgs a = {};
  a.x = x, a.x_sb = x_sb, a.x_st = x_st, a.w = w, a.bias = bias, a.init = init, a.len = len;
  a.y = y, a.final_state = final_state, a.T = T, a.C = C, a.silu = silu;
  a.run = run_of(B, T, C, false), a.ygrid = ygrid_of(T, a.run);
  cudaStream_t st = (cudaStream_t)stream;
  return dtype_io == ATLAS_BF16 ? dispatch<__nv_bfloat16>(true, K, a, B, nullptr, nullptr, st)
                                : dispatch<float>(true, K, a, B, nullptr, nullptr, st);
}

size_t atlas_causal_conv_scratch(int64_t B, int64_t T, int64_t C, int K) {
  if (!shape_ok(K, ATLAS_F32, B, T, C)) return 0;
  return (size_t)B * ygrid_of(T, run_of(B, T, C, true)) * C * (K + 1) * sizeof(float);
}

int atlas_causal_conv_backward(const void* x, int64_t x_sb, int64_t x_st, const float* w, const float* bias,
                               const void* init, const int32_t* len, const void* dy, int64_t dy_sb, int64_t dy_st,
                               const void* d_final, void* dx, void* d_init, float* dw, float* dbias, void* scratch,
                               size_t scratch_bytes, int K, int silu, int dtype_io, int64_t B, int64_t T, int64_t C,
                               void* stream) {
  if (!x || !w || !dy || !dx || !dw || !shape_ok(K, dtype_io, B, T, C)) return ATLAS_ERR_INVALID_ARG;
  if (!scratch || scratch_bytes < atlas_causal_conv_scratch(B, T, C, K)) return ATLAS_ERR_WORKSPACE;
  ConvArgs a = {};
  a.x = x, a.x_sb = x_sb, a.x_st = x_st, a.w = w, a.bias = bias, a.init = init, a.len = len;
  a.dy = dy, a.dy_sb = dy_sb, a.dy_st = dy_st, a.d_final = d_final, a.dx = dx, a.d_init = d_init;
  a.part = (float*)scratch, a.T = T, a.C = C, a.silu = silu;
  a.run = run_of(B, T, C, true), a.ygrid = ygrid_of(T, a.run);
  cudaStream_t st = (cudaStream_t)stream;
  return dtype_io == ATLAS_BF16 ? dispatch<__nv_bfloat16>(false, K, a, B, dw, dbias, st)
                                : dispatch<float>(false, K, a, B, dw, dbias, st);
}

}  // extern "C"
