// sd_paged_inst.cu -- instantiates the paged decode kernels of one storage
// format; compiled once per (SD_E, SD_BITS) pair like sd_inst.cu.
#include "sd_paged.cuh"

#if !defined(SD_E) || !defined(SD_BITS)
#error "SD_E and SD_BITS must be defined"
#endif

#if SD_E == 0
using ET = float;
#elif SD_E == 1
using ET = __half;
#else
using ET = __nv_bfloat16;
#endif

#define SD_NAME2(e, b) paged_e##e##_b##b
#define SD_NAME(e, b) SD_NAME2(e, b)

namespace sd {

template <int D, int NB>
static PagedSet make_paged() {
  using F = PagedFmt<sizeof(ET), SD_BITS, D>;
  PagedSet s;
  s.decode = reinterpret_cast<const void*>(&paged_decode_kernel<ET, SD_BITS, D, NB>);
  s.merge = reinterpret_cast<const void*>(&paged_merge_kernel<ET, D, F::kTile, 1>);
  s.merge_many = reinterpret_cast<const void*>(&paged_merge_kernel<ET, D, F::kTile, kMergeHeads>);
  s.tile = F::kTile;
  s.stage_bytes = F::kStageBytes;
  return s;
}

template <int D>
static PagedSet pick_heads(int G) {
#if SD_E == 0 && SD_BITS == 0
  return G <= 4 ? make_paged<D, 1>() : G <= 8 ? make_paged<D, 2>() : make_paged<D, 4>();  // blocks of 4 heads
#else
  return G <= 8 ? make_paged<D, 1>() : make_paged<D, 2>();  // blocks of 8
#endif
}

PagedSet SD_NAME(SD_E, SD_BITS)(int D, int G) {
  return D == 64 ? pick_heads<64>(G) : D == 128 ? pick_heads<128>(G) : PagedSet{};
}

}  // namespace sd
