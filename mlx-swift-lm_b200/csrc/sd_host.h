// sd_host.h -- host-side helpers shared by the C ABI's source files.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace sd {

// Keep the message for sd_last_error on this thread and return `status`.
int32_t fail(int32_t status, const char* fmt, ...);

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn();

// Tensor map of `rows` rows of row_bytes at `base`, copied box_rows rows at a time.
int32_t encode_map(CUtensorMap* map, void* base, int row_bytes, int64_t rows, int box_rows);

}  // namespace sd

#define SD_CUDA(call)                                                                                    \
  do {                                                                                                   \
    cudaError_t e_ = (call);                                                                             \
    if (e_ != cudaSuccess) return sd::fail(SD_ERR_CUDA, "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), \
                                           __FILE__, __LINE__);                                          \
  } while (0)
