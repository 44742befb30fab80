// Launch accounting shared by the library's translation units: every kernel has an id and a
// name, every launch is counted, and with timing on (atlas_mem_profile_enable) it is bracketed
// by CUDA events on its own stream. Defined in atlas_mem.cu.
#pragma once
#include <cuda_runtime.h>

#include "atlas_mem.h"

namespace atlas {

enum KernelId {
  KID_FMAP_FWD, KID_FWD_CHUNK, KID_FWD_SCAN, KID_FWD_OUT, KID_BUF_OUT, KID_BWD_CHUNK, KID_BWD_SCAN,
  KID_BWD_GRADS, KID_BWD_BUFOUT, KID_BWD_FINAL, KID_BWD_DSREF, KID_FMAP_BWD, KID_FWD_CHUNK_TC, KID_FWD_OUT_TC, KID_FWD_BUF_Y,
  KID_BWD_CHUNK_TC, KID_BWD_STATE_GATES_TC, KID_BWD_BUF_TC, KID_BWD_FINAL_TC, KID_BWD_DSREF_TC, KID_BWD_KEYS_TC, KID_SREF_TILE, KID_DECODE, KID_SCAN_OP_FWD, KID_SCAN_OP_BWD, KID_CARRY, KID_DWCONV_FWD, KID_DWCONV_BWD, KID_HEADPREP_FWD, KID_HEADPREP_BWD, KID_PROJ_TILES, KID_FMAP_FWD_TC, KID_FMAP_BWD_TC, KID_OMEGA_STORE_FWD, KID_OMEGA_STORE_BWD, KID_AFFINE_FWD, KID_AFFINE_BWD,
  KID_SSCAN_FWD, KID_SSCAN_ENDS, KID_SSCAN_CARRY, KID_SSCAN_STEP, KID_SSCAN_BWD, KID_SSCAN_BWD_ENDS, KID_SSCAN_DBC, KID_SSCAN_DA,
  KID_CONV_FWD, KID_CONV_STEP, KID_CONV_BWD, KID_CONV_DW, KID_SAMPLE, KID_DISTILL_FWD, KID_DISTILL_BWD, KID_COUNT
};

int prof_begin(int kid, cudaStream_t st);
void prof_end(int slot, cudaStream_t st);
int sm_count();  // multiprocessors of the current device

}  // namespace atlas

#define LAUNCH_CHECK()                                              \
  do {                                                              \
    if (cudaGetLastError() != cudaSuccess) return ATLAS_ERR_LAUNCH; \
  } while (0)

// Launch with an explicit thread count: LAUNCH_T(id, kernel, grid, threads, smem, stream, args...)
#define LAUNCH_T(KID, KERNEL, GRID, THREADS, SMEM, STREAM, ...)   \
  do {                                                            \
    const int slot_ = prof_begin(KID, STREAM);                    \
    KERNEL<<<GRID, THREADS, SMEM, STREAM>>>(__VA_ARGS__);         \
    LAUNCH_CHECK();                                               \
    prof_end(slot_, STREAM);                                      \
  } while (0)

// Launch `kernel` with accounting: LAUNCH(id, kernel, grid, smem, stream, args...)
#define LAUNCH(KID, KERNEL, GRID, SMEM, STREAM, ...)              \
  do {                                                            \
    const int slot_ = prof_begin(KID, STREAM);                    \
    KERNEL<<<GRID, kThreads, SMEM, STREAM>>>(__VA_ARGS__);        \
    LAUNCH_CHECK();                                               \
    prof_end(slot_, STREAM);                                      \
  } while (0)
