// sd_pages_host.h -- host helpers of the paged operators' C ABI: checks of a
// pool, where its arrays lie, launches.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "../../include/sparse_decode.h"
#include "sd_host.h"

namespace sd {

inline int elt_size(int dtype) { return dtype == SD_F32 ? 4 : 2; }
inline bool misaligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }
inline int log2_of(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}

inline int32_t check_dtype(int32_t dtype) {
  if (dtype != SD_F32 && dtype != SD_F16 && dtype != SD_BF16) return fail(SD_ERR_INVALID_ARG, "unknown dtype %d", dtype);
  return SD_OK;
}

// Everything about a pool that can be checked on the host.
inline int32_t check_pages(const sd_pages* g) {
  if (!g) return fail(SD_ERR_INVALID_ARG, "pages is NULL");
  if (int32_t rc = check_dtype(g->dtype)) return rc;
  if (g->n_pages < 1 || g->n_layers < 1 || g->n_kv_heads < 1)
    return fail(SD_ERR_INVALID_ARG, "n_pages, n_layers and n_kv_heads must be positive");
  if (g->head_dim != 64 && g->head_dim != 128) return fail(SD_ERR_SHAPE, "head_dim must be 64 or 128 (got %d)", g->head_dim);
  const int P = g->page_size;
  if (P != 16 && P != 32 && P != 64 && P != 128 && P != 256)
    return fail(SD_ERR_SHAPE, "page_size must be 16, 32, 64, 128 or 256 (got %d)", P);
  if (g->kv_bits != 0 && g->kv_bits != 4 && g->kv_bits != 8)
    return fail(SD_ERR_SHAPE, "kv_bits must be 0, 4 or 8 (got %d)", g->kv_bits);
  if (g->group_size != (g->kv_bits ? 64 : 0))
    return fail(SD_ERR_SHAPE, "group_size must be 64 for quantized pools and 0 for dense ones");
  if (g->reserved != 0) return fail(SD_ERR_INVALID_ARG, "reserved fields must be 0");
  if (g->n_pages > (int64_t(1) << 31) || g->n_pages * g->n_kv_heads >= (int64_t(1) << 31) / P)
    return fail(SD_ERR_SHAPE, "pool too large: n_pages * n_kv_heads * page_size rows must stay below 2^31");
  const void* a[6] = {g->k_data, g->v_data, g->k_scales, g->k_biases, g->v_scales, g->v_biases};
  for (int i = 0; i < (g->kv_bits ? 6 : 2); ++i) {
    if (!a[i]) return fail(SD_ERR_INVALID_ARG, "a pool array is NULL");
    if (misaligned(a[i], 16)) return fail(SD_ERR_INVALID_ARG, "pool arrays must be 16-byte aligned");
  }
  return SD_OK;
}

inline int32_t check_layer(const sd_pages* g, int32_t layer) {
  if (layer < 0 || layer >= g->n_layers) return fail(SD_ERR_INVALID_ARG, "layer %d out of range", layer);
  return SD_OK;
}

inline int row_bytes(const sd_pages* g) {
  return g->kv_bits ? g->head_dim * g->kv_bits / 8 : g->head_dim * elt_size(g->dtype);
}
inline int sb_bytes(const sd_pages* g) { return g->kv_bits ? g->head_dim / 64 * elt_size(g->dtype) : 0; }
inline int64_t layer_rows(const sd_pages* g) { return g->n_pages * g->n_kv_heads * g->page_size; }
inline void* at(void* base, int64_t bytes) { return base ? static_cast<uint8_t*>(base) + bytes : nullptr; }

inline int32_t sm_count(int* n) {
  static std::atomic<int> known[64];
  int dev = 0;
  SD_CUDA(cudaGetDevice(&dev));
  int v = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (v == 0) {
    SD_CUDA(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) known[dev].store(v, std::memory_order_relaxed);
  }
  *n = v;
  return SD_OK;
}

// The launches here may begin while the kernel before them on the stream
// ends (programmatic dependent launch); every kernel waits for it
// (griddepcontrol.wait) before its first access to memory, and lets its own
// successor begin only after that, so that whatever begins early finds all
// work before its predecessor complete. One access comes before the wait: the
// merge reads the lengths, which no decode kernel writes and whatever did is
// complete. Since a kernel's inputs may be written
// while it already waits, none is read through the non-coherent path.
inline int32_t launch(const void* fn, dim3 grid, int threads, size_t smem, cudaStream_t st, void** args, int cluster = 1) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  SD_CUDA(cudaLaunchKernelExC(&cfg, fn, args));
  return SD_OK;
}

}  // namespace sd
