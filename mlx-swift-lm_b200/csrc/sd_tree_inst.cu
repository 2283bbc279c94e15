// sd_tree_inst.cu -- instantiates the tree attention kernels of one storage
// format; compiled once per (SD_E, SD_BITS) pair like sd_paged_inst.cu.
#include "sd_tree.cuh"

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

#define SD_NAME2(e, b) tree_e##e##_b##b
#define SD_NAME(e, b) SD_NAME2(e, b)

namespace sd {

template <int D, int NB>
static TreeSet make_tree() {
  using F = PagedFmt<sizeof(ET), SD_BITS, D>;
  TreeSet s;
  s.attend[0] = reinterpret_cast<const void*>(&tree_attend_kernel<ET, SD_BITS, D, NB, false>);
  s.attend[1] = reinterpret_cast<const void*>(&tree_attend_kernel<ET, SD_BITS, D, NB, true>);
  s.merge = reinterpret_cast<const void*>(&tree_merge_kernel<ET, D>);
  s.tile = F::kTile;
  s.stage_bytes = F::kStageBytes;
  s.columns = NB * (SD_E == 0 && SD_BITS == 0 ? 4 : 8);
  return s;
}

template <int D>
static TreeSet pick_columns(int columns) {
#if SD_E == 0 && SD_BITS == 0
  return columns <= 4 ? make_tree<D, 1>() : columns <= 8 ? make_tree<D, 2>() : make_tree<D, 4>();  // blocks of 4
#else
  return columns <= 8 ? make_tree<D, 1>() : make_tree<D, 2>();  // blocks of 8
#endif
}

TreeSet SD_NAME(SD_E, SD_BITS)(int D, int columns) {
  return D == 64 ? pick_columns<64>(columns) : D == 128 ? pick_columns<128>(columns) : TreeSet{};
}

}  // namespace sd
