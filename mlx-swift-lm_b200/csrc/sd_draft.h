// sd_draft.h -- parameters and kernels of the operators around drafted tokens:
// the plan of a step, the rows that are kept, attention over trees. Included by
// host and device code.
#pragma once

#include <cuda_runtime.h>

#include "sd_paged.h"

namespace sd {

constexpr int kMaxNodes = 64;  // new tokens of one sequence in a tree: the bits of a mask

// ---------------------------------------------------------------------------
// The plan of a step and the rows that are kept
// ---------------------------------------------------------------------------

constexpr int kPlanThreads = 256;
constexpr int kPlanRows = 4;      // rows that a thread takes at a time: 16-byte stores
constexpr int kPlanCluster = 8;   // CTAs that may wait for one another

struct PlanParams {
  const int *lengths, *added;  // [B]
  int* tables;                 // [B, W]
  int* held;                   // [B] or null: no pages are taken
  const int* free_pages;
  int* taken;
  const int* parents;          // [B or 1, T] or null
  int64_t parents_stride;      // of a sequence; 0: one tree for all
  int n_free, T;
  int B, W, P, page_shift, N;
  int *first, *ends, *seq, *positions, *places;
  int64_t *slots, *masks;
  int* flags;
  bool rows, commit;           // what this launch does: the rows, the pages taken
};
// Dynamic shared memory of a plan launch: rows before, lengths, held pages and pages before each sequence.
constexpr int plan_smem(int B) { return (4 * B + 1) * 4; }
const void* plan_kernel_ptr();

struct KeepParams {
  const int *tables, *ends, *first, *path, *kept;
  int* lengths;
  int B, W, P, page_shift, N, T, Hkv;
  int64_t n_pages;
  uint8_t* array[6];
  int row[6];                 // bytes of a row (token and head) in each array
  int64_t layer[6];           // bytes of a layer
  int columns[6];             // accesses that make one token's rows of each array: heads * row / width
  int all_columns;
  int* flags;
};
constexpr int kKeepThreads = 256;
constexpr int kKeepBatch = 8;  // rows that a thread has under way
const void* keep_kernel_ptr();

// ---------------------------------------------------------------------------
// Attention over trees
// ---------------------------------------------------------------------------

// lengths: tokens of each sequence, its new ones counted in; G, q and out: of packed rows [N, Hq, D].
struct TreeParams : PagedParams {
  const int* first;        // [B + 1]
  const int64_t* masks;    // [N] or null: a node sees those up to itself
  const int* places;       // [N] or null: the position of each node, for windows
  const uint8_t *k_data, *v_data;  // of this layer
  int* line;               // [2][B + 1]: units and pairs before each sequence
  int N, Hq;
  int seg_units;           // see tree_units
  int raw_stages;          // of the tile kernel for codes
  int RT;                  // columns (node, query head) of a pair
  int part_floats;         // of one segment in the workspace: o [D / 4][RT][4], then (m, l) [RT]
  float* node_o;           // [N * Hq][D], of the nodes alone
  float2* node_ml;         // [N * Hq]; null: the nodes are on the line
  FastDiv by_g;            // G
};

struct TreeSet {
  const void* attend[2];  // tree_attend_kernel<E, BITS, D, blocks of columns, help>(TreeParams, CUtensorMap, CUtensorMap)
  const void* merge;      // tree_merge_kernel<E, D>(TreeParams)
  int tile, stage_bytes, columns;
};
// For at most `columns` columns a pair, or as many as there are.
TreeSet tree_e0_b0(int D, int columns);
TreeSet tree_e1_b0(int D, int columns);
TreeSet tree_e2_b0(int D, int columns);
TreeSet tree_e0_b4(int D, int columns);
TreeSet tree_e1_b4(int D, int columns);
TreeSet tree_e2_b4(int D, int columns);
TreeSet tree_e0_b8(int D, int columns);
TreeSet tree_e1_b8(int D, int columns);
TreeSet tree_e2_b8(int D, int columns);

constexpr int kTreeHeads = 4;      // query heads that a warp takes to the nodes at once
constexpr int kTreeAttendThreads = kPagedThreads + 32;  // a decode's, and a warp for the nodes
constexpr int kTreeMergeCols = 8;  // columns of a merge block

// Shared memory of an attend CTA: as a decode's, with two numbers per sequence and per warp, the columns' first tokens and
// two counts (tree_attend_kernel: units, pairs, tmp, low, next).
constexpr int kTreeLows = 16, kTreeCounts = 2;
constexpr int tree_attend_ints(int batch) { return 2 * (batch + 1) + 2 * (kTreeAttendThreads / 32) + kTreeLows + kTreeCounts; }
constexpr PagedLayout tree_layout(int batch, int columns, int D, bool dense_f32, int stage_bytes) {
  return paged_layout_of(tree_attend_ints(batch) * 4, columns, D, dense_f32, stage_bytes);
}

// The tile kernel of 16-bit pools (sd_tree_tile.cu): one CTA per SM, two groups
// of four warps, a warp that issues products for each and a loading warp.
// The rule for it: more columns, of an average sequence, than tree_attend_kernel has in one pass over the tokens, or in two
// of codes. Measured with 8 sequences of 8K tokens and 8 kv heads, us, that kernel and this one: bf16, heads of 128, 16
// columns 50 and 60, 20 columns 88 and 61; of 64, 16 columns 31 and 48, 20 columns 50 and 48. 4 bits, heads of 128, 32 columns
// 89 and 114, 40 columns 124 and 114, 64 columns 164 and 118, 128 columns 323 and 125; of 64, 40 columns 70 and 88, 64
// columns 90 and 89, 128 columns 169 and 91; 8 bits the same within 6 us. 16 sequences of 700 tokens, 4 bits, heads of 128, 32
// columns 45 and 42, 40 columns 70 and 45; of 64, 40 columns 35 and 32.
constexpr int tree_tile_above(int bits) { return bits ? 32 : 16; }
constexpr int kTreeTileThreads = 352;
constexpr int kTreeTileTokens = 64;
// Beginning and ending a segment, in tiles. Measured, 2 / 4 / 8 / 16: 12 windows of 1000 tokens, 168 columns, 41.6 / 32.7 /
// 30.9 / 30.5 us; 16 ragged sequences of about 4K, 64 columns, plan to keep, 78 / 60 / 52 / 60 us; one of 32K, 128 columns,
// 43.2 / 41.8 / 39.9 / 40.3 us; 4 x 32K in 4 bits 199 / 199 / 200 / 203 us.
constexpr int kTreeTileUnits = 8;
constexpr int kTreeTileStages = 24, kTreeTileLeast = 4;
constexpr int kTreeTileBarBytes = 768;
// For codes eight more warps make tiles of values of them, in two halves each.
constexpr int kTreeCodeThreads = 640;
constexpr int kTreeRawStages = 8;
__host__ __device__ constexpr int tree_tile_queries(int D, int bits, bool shared) { return bits && !shared && D == 128 ? 1 : 2; }
// Codes of K and V of a tile and their scales and biases.
__host__ __device__ constexpr int tree_raw_stage(int D, int bits) {
  return bits ? 2 * kTreeTileTokens * D * bits / 8 + 4 * kTreeTileTokens * (D / 64) * 2 : 0;
}
constexpr int kTreeTileSmem = 232448 - 4096;  // beside 4 KB of static shared memory
// For rows of `shared`: up to 256 columns, not for codes, else up to 128 (both groups hold them all).
const void* tree_tile_e1_b0(int D, bool shared);
const void* tree_tile_e2_b0(int D, bool shared);
const void* tree_tile_e2_b4(int D, bool shared);
const void* tree_tile_e2_b8(int D, bool shared);

struct TileLayout {
  int stages, raw_stages;
  int raw_off, prefix_off, bar_off, bytes;
};
constexpr TileLayout tree_tile_layout(int batch, int D, int bits, bool shared) {
  const int stage = kTreeTileTokens * D * 2, q = tree_tile_queries(D, bits, shared) * 128 * D * 2, raw = tree_raw_stage(D, bits);
  const int pre = (2 * (batch + 1) + 2 * (kTreeCodeThreads / 32)) * 4, pre128 = (pre + 127) / 128 * 128;
  int room = kTreeTileSmem - 1024 - q - pre128 - kTreeTileBarBytes;
  TileLayout l{};
  // Where the groups take tiles in turn, a stage stays with the K, or the V, of one of them: a wait for a stage names
  // its phase by the parity, so whoever waits has to know that the phase before is done.
  // (Of codes, with one of the two teams of warps that make the tiles, too.)
  const int by = shared && !bits ? 1 : 4;
  if (bits) {  // eight tiles of halves of values, or four, and the rest for codes, but two stages at least
    const int fit = (room - 2 * raw) / stage;
    l.stages = (fit < 8 ? fit : 8) / by * by;
    l.raw_stages = (room - l.stages * stage) / raw / 2 * 2;
    if (l.raw_stages > kTreeRawStages) l.raw_stages = kTreeRawStages;
  } else {
    l.stages = room / stage;
    if (l.stages > kTreeTileStages) l.stages = kTreeTileStages;
    l.stages = l.stages / by * by;
  }
  l.raw_off = q + l.stages * stage;
  l.prefix_off = (l.raw_off + l.raw_stages * raw + 127) / 128 * 128;
  l.bar_off = l.prefix_off + pre128;
  l.bytes = l.bar_off + kTreeTileBarBytes + 1024;
  return l;
}

}  // namespace sd
