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
  s.merge = reinterpret_cast<const void*>(&paged_merge_kernel<ET, D, F::kTile>);
  s.tile = F::kTile;
  s.stage_bytes = F::kStageBytes;
  s.row_bytes = F::kRowBytes;
  s.groups = F::kGroups;
  return s;
}

PagedSet SD_NAME(SD_E, SD_BITS)(int D, int nb) {
  if (D == 64) return nb == 1 ? make_paged<64, 1>() : make_paged<64, 2>();
  if (D == 128) return nb == 1 ? make_paged<128, 1>() : make_paged<128, 2>();
  return PagedSet{nullptr, nullptr, 0, 0, 0, 0};
}

}  // namespace sd
