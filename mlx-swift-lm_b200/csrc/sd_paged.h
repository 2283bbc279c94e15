// sd_paged.h -- parameters, launch shapes and kernel tables of the operators
// on a paged KV pool: decode attention, append (with rotation) and page
// copies. Included by host and device code.
#pragma once

#include <stdint.h>

#include "sd_format.h"

namespace sd {

constexpr int kPagedWarps = 4;                          // warps that attend
constexpr int kPagedThreads = (kPagedWarps + 1) * 32;   // + one producer warp
constexpr int kMergeThreads = 256;
// Query heads of one merge block in calls of more than kMergeMany (sequence,
// query head) pairs, which come in several waves as blocks of one head each:
// 39 ragged sequences to 2.6K tokens, 128 heads on 4-bit codes 71 -> 49 us, 16
// sequences of 2K, 32 heads in bf16 29.5 -> 27.4; at 256 pairs and below blocks
// of one head are as fast, or faster where a sequence has many segments (4
// ragged sequences to 60K, 32 heads 67.5, 69.2 by eight).
constexpr int kMergeHeads = 8, kMergeMany = 256;
constexpr int kPagedMaxBatch = 4096;                    // sequences per decode call
constexpr int kPagedMaxStages = 16;
// Beginning and ending a segment costs about as much as two tiles. With 16
// ragged users of up to 4096 tokens in 8 bits, a decode took 25.2 us when cut
// by tiles alone, 19.9 / 19.3 / 20.2 us with 1 / 2 / 3.
constexpr int kSegmentUnits = 2;
// Two CTAs share an SM: half of its 228 KB each, less 1 KB that every CTA
// reserves. All of it is dynamic: 32 static bytes beside a full dynamic share
// left room for one CTA only, and the second half of the grid ran after the
// first (11 heads of 64 per kv head on 4-bit codes, 4 x 32K tokens: 66.2 us,
// 44.3 without them; 224 bf16 sequences of 2K, 28 heads: 150.8, 147.2).
constexpr int kPagedSmem = 115712;

// Stored rows of one pool format: E of ESIZE bytes (dense element, or type of
// the scales and biases), BITS = 0 / 4 / 8.
template <int ESIZE, int BITS, int D>
struct PagedFmt {
  static constexpr int kRowBytes = BITS ? D * BITS / 8 : D * ESIZE;
  static constexpr int kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;
  static constexpr int kNBox = kRowBytes / kBoxBytes;
  static constexpr int kCpb = kBoxBytes / 16;           // 16-byte chunks per box row
  static constexpr int kNChunk = kRowBytes / 16;
  static constexpr int kEpc = BITS ? 128 / BITS : 16 / ESIZE;  // elements per chunk
  static constexpr int kGroups = BITS ? D / 64 : 1;
  // Tokens of one stage. Codes take 32 tokens per warp (two m-tiles), so that
  // what a tile costs beside its tokens weighs less: 4 x 128K tokens in 8 bits
  // 178 us, 218 us with 64 tokens per tile. 16-bit rows are bound by the loads
  // with 16 per warp already; dense fp32 warps hold 8 tokens.
  static constexpr int kTile = ESIZE == 4 ? (BITS ? 64 : 32) : BITS ? 128 : 64;
  static constexpr int kKvBytes = kTile * kRowBytes;    // K (or V) of a stage
  static constexpr int kSbBytes = BITS ? kTile * kGroups * ESIZE : 0;  // each of the four scale/bias pieces
  static constexpr int kStageBytes = (2 * kKvBytes + 4 * kSbBytes + 1023) / 1024 * 1024;
};

// Floats of one warp's (o, m, l) in the combine buffer -- o rows padded to
// D + 4, which spreads the fragment stores over the banks -- and of one
// unfinished segment in the workspace; multiples of 4, as both are read with
// 16-byte accesses.
__host__ __device__ constexpr int paged_warp_floats(int G, int D) { return (G * (D + 6) + 3) / 4 * 4; }
__host__ __device__ constexpr int paged_part_floats(int G, int D) { return (G * (D + 2) + 3) / 4 * 4; }

// Where the parts of a decode CTA's shared memory lie, from a 1 KB boundary:
// the ring, q of dense fp32 calls, the warps' combine buffer, the units before
// each sequence (and the warps' totals of them), the ring's barriers.
struct PagedLayout {
  int stages;  // as many as fit beside the fixed parts; below 1: the call does not fit
  int q_off, buf_off, prefix_off, bar_off;
  int bytes;   // of the launch, the way to the boundary included
};
constexpr PagedLayout paged_layout_of(int pre, int G, int D, bool dense_f32, int stage_bytes) {  // pre: bytes
  const int qf = dense_f32 ? G * (D + 4) * 4 : 0, buf = kPagedWarps * paged_warp_floats(G, D) * 4;
  const int bars = 2 * kPagedMaxStages * 8;
  const int q128 = (qf + 127) / 128 * 128, buf128 = (buf + 127) / 128 * 128, pre128 = (pre + 127) / 128 * 128;
  const int room = (kPagedSmem - (q128 + buf128 + pre128 + bars + 1024)) / stage_bytes;
  PagedLayout l{};
  l.stages = room < kPagedMaxStages ? room : kPagedMaxStages;
  l.q_off = l.stages * stage_bytes;
  l.buf_off = l.q_off + q128;
  l.prefix_off = l.buf_off + buf128;
  l.bar_off = l.prefix_off + pre128;
  l.bytes = l.bar_off + bars + 1024;
  return l;
}
constexpr PagedLayout paged_layout(int batch, int G, int D, bool dense_f32, int stage_bytes) {
  // below 32 sequences every warp has its own row of 32
  const int pre = (batch < 32 ? 32 * (kPagedWarps + 1) : batch + 1 + kPagedThreads / 32) * 4;
  return paged_layout_of(pre, G, D, dense_f32, stage_bytes);
}

struct PagedParams {
  const void* q;          // [B, Hkv * G, D]
  void* out;              // [B, Hkv * G, D]
  float* part;            // [grid][2][paged_part_floats]: o [G][D], then (m, l) [G]
  const int* tables;      // [B, W]
  const int* lengths;     // [B]
  const float* sinks;     // [Hkv * G] or null
  const void *k_scales, *k_biases, *v_scales, *v_biases;  // of this layer
  int64_t n_pages;
  int B, Hkv, G, P, W, window;
  int stages, ncta;
  int q_off, buf_off, prefix_off, bar_off;  // shared-memory layout
  float scale_log2;
  uint32_t magic;         // 0x64006400, see raw_u8
  int* flags;
};

struct PagedSet {
  const void* decode;  // paged_decode_kernel<E, BITS, D, blocks of heads>(PagedParams, CUtensorMap, CUtensorMap)
  const void *merge, *merge_many;  // paged_merge_kernel<E, D, tile, 1 or kMergeHeads>(PagedParams)
  int tile, stage_bytes;
};
// For G query heads per kv head; null members without an instantiation.
PagedSet paged_e0_b0(int D, int G);
PagedSet paged_e1_b0(int D, int G);
PagedSet paged_e2_b0(int D, int G);
PagedSet paged_e0_b4(int D, int G);
PagedSet paged_e1_b4(int D, int G);
PagedSet paged_e2_b4(int D, int G);
PagedSet paged_e0_b8(int D, int G);
PagedSet paged_e1_b8(int D, int G);
PagedSet paged_e2_b8(int D, int G);

// ---------------------------------------------------------------------------

// n / d for 0 <= n < 2^31 by a multiplication: a hardware division costs tens
// of instructions, and the row kernels would make several per row.
struct FastDiv {
  uint32_t mul, shift;
  int d;
  void set(int div) {
    d = div;
    shift = 0;
    while ((uint64_t(1) << shift) < uint64_t(div)) ++shift;
    mul = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - uint64_t(div))) / uint64_t(div) + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int operator()(int n) const { return int((__umulhi(uint32_t(n), mul) + uint32_t(n)) >> shift); }
#endif
};

// Rows [batch, tokens, heads, D] with D contiguous; strides in elements.
struct Rows {
  void* data;
  int64_t batch, token, head;
};

struct RotaryParams {
  Rows q, k, v, q_out, k_out;
  int Hq, Hkv, Hv;          // heads of q, k and v rows per token (0: none)
  int D, rot2;              // head_dim, rotated pairs (0: no rotation)
  float inv_dim;            // 1 / D
  FastDiv L;                // tokens per batch entry
  FastDiv pairs;            // rot2
  int n_tokens;             // batch * L
  // The warps of each kind of rows (queries, keys, values): a warp takes
  // 2^tok_log tokens and makes `span` of the passes over their heads.
  struct Kind {
    int first;              // first warp
    int tok_log;
    int span;               // passes that one warp makes
    FastDiv per;            // warps per group of tokens
  } kind[3];
  int units;                // warps in all
  int ring_at;              // byte offset of the row ring in shared memory
  const int* positions;     // [batch * L]
  const float* inv_freq;    // [rot2]
  const void *q_norm, *k_norm;
  float eps, factor;
  // append: where the k and v rows go (null tables: k_out)
  const int* tables;
  const int* seq;
  int B, W, P, page_shift;
  int64_t n_pages;
  void *k_data, *v_data, *k_scales, *k_biases, *v_scales, *v_biases;
  int* flags;
};

constexpr int kRotThreads = 128;
// Measured on a 32K-token prompt of 32 + 8 heads of 128 (671 MB, floor 102 us)
// and, for kRotFill, on 1000 tokens of it:
constexpr int kRotDepth = 4;          // passes whose rows are under way: 107 us; 3: 114, 6: 112
constexpr int kRotPasses = 16;        // most passes that one warp makes: 107.5 us; 8: 108.2, 32: 110.5
constexpr int kRotFill = 2048;        // warps that fill the GPU: 6.2 us; 1024: 7.3, 4096: 7.4
// Lanes per row (log2): a power of two with a chunk pair of 2 * vec elements for each, at most a warp.
__host__ __device__ constexpr int rotary_lanes_log(int D, int vec) {
  int l = 0;
  while (l < 5 && (1 << l) < D / (2 * vec)) ++l;
  return l;
}
// Floats of a cos (or sin) row in shared memory: whole 16-byte pieces.
__host__ __device__ constexpr int rotary_pitch(int rot2) { return (rot2 + 7) / 8 * 8; }

// vec: elements per access (1, 2, 4, and 8 for 16-bit types); wide: head_dim
// above 128; shifted: rotated halves that are no whole number of accesses (vec
// is 4 then).
const void* rotary_kernel_for(int dtype, int bits, int vec, bool wide, bool shifted, bool traditional);

struct CopyParams {
  const int *src, *dst;
  int n;
  int64_t n_pages;
  uint8_t* array[6];
  int64_t bytes[6];   // of one page in each array
  int pieces[6];      // kCopyPiece pieces of one page
  int per_pair;       // pieces of one page pair in one layer
  int* flags;
};
constexpr int kCopyPiece = 32768;
constexpr int kCopyThreads = 256;
const void* copy_pages_kernel_ptr();

}  // namespace sd
