// sd_steps.cu -- the C ABI of the operators around drafted tokens: argument
// checks, launch shapes and launches (kernels in sd_draft.cu, sd_tree.cuh).
// Host code only.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <utility>

#include "sd_draft.h"
#include "sd_pages_host.h"

namespace {

using namespace sd;

static_assert(SD_MAX_NODES == kMaxNodes, "the bits of a mask");

TreeSet lookup_tree(int dtype, int bits, int D, int columns) {
  switch (dtype * 16 + bits) {
    case 0 * 16 + 0: return tree_e0_b0(D, columns);
    case 1 * 16 + 0: return tree_e1_b0(D, columns);
    case 2 * 16 + 0: return tree_e2_b0(D, columns);
    case 0 * 16 + 4: return tree_e0_b4(D, columns);
    case 1 * 16 + 4: return tree_e1_b4(D, columns);
    case 2 * 16 + 4: return tree_e2_b4(D, columns);
    case 0 * 16 + 8: return tree_e0_b8(D, columns);
    case 1 * 16 + 8: return tree_e1_b8(D, columns);
    case 2 * 16 + 8: return tree_e2_b8(D, columns);
    default: return TreeSet{};
  }
}

const void* (*lookup_tile(int dtype, int bits))(int, bool) {
  if (dtype == SD_F16) return bits == 0 ? tree_tile_e1_b0 : nullptr;
  if (dtype != SD_BF16) return nullptr;
  return bits == 0 ? tree_tile_e2_b0 : bits == 4 ? tree_tile_e2_b4 : tree_tile_e2_b8;
}

bool good_page(int P) { return P == 16 || P == 32 || P == 64 || P == 128 || P == 256; }

bool any_misaligned4(std::initializer_list<const void*> list) {
  for (const void* x : list)
    if (misaligned(x, 4)) return true;
  return false;
}

// How a call is cut: by the rows of an average sequence, as the host knows no more.
struct TreeShape {
  const void* attend;
  const void* merge;
  int threads, smem_most;  // of attend
  TileLayout lay;
  int q_off, buf_off;
  int tile, columns;  // tokens of a tile, columns of a pair
  bool tiles;         // the tile kernel
  int ctas, seg_units;
  int64_t pairs;      // at most
  int part_floats;
  int64_t line_bytes, node_bytes, bytes;  // of the workspace: line, segments, the nodes' (m, l) and o
};

int32_t tree_shape(const sd_pages* g, int32_t batch, int32_t n_rows, int32_t n_q_heads, TreeShape* s) {
  const int G = n_q_heads / g->n_kv_heads, D = g->head_dim;
  const int64_t columns = (int64_t(n_rows) + batch - 1) / batch * G;
  int sms = 0;
  if (int32_t rc = sm_count(&sms)) return rc;
  const TreeSet set = lookup_tree(g->dtype, g->kv_bits, D, int(std::min<int64_t>(columns, 16)));
  if (!set.merge) return fail(SD_ERR_SHAPE, "no kernel for dtype %d, bits %d, head_dim %d", g->dtype, g->kv_bits, D);
  s->merge = set.merge;
  // Codes of fp16 pools are not for the tile kernel: its tiles of them, two bf16 values each, would need queries in two
  // as well.
  const auto tile_kernel = lookup_tile(g->dtype, g->kv_bits);
  const bool shared = columns > 128 && !g->kv_bits;
  s->lay = tree_tile_layout(batch, D, g->kv_bits, shared);
  // Of codes a tile of K or V is two, of high and low halves, and two tiles are under way: thousands of sequences with heads
  // of 128 leave no room for that in 8 bits.
  s->tiles = tile_kernel && columns > tree_tile_above(g->kv_bits) && (!g->kv_bits || s->lay.stages == 8);
  if (s->tiles) {
    s->attend = tile_kernel(D, shared);
    s->threads = g->kv_bits ? kTreeCodeThreads : kTreeTileThreads;
    s->smem_most = kTreeTileSmem;
    s->q_off = s->lay.raw_off;
    if (g->kv_bits) s->lay.stages /= 2;
    s->tile = kTreeTileTokens;
    s->columns = shared ? 256 : 128;
    s->ctas = sms;
    s->seg_units = kTreeTileUnits;
  } else {
    s->ctas = 2 * sms;
    s->attend = set.attend[int64_t(n_rows) * g->n_kv_heads * ((G + kTreeHeads - 1) / kTreeHeads) > s->ctas];
    s->threads = kTreeAttendThreads;
    s->smem_most = kPagedSmem;
    const PagedLayout lay = tree_layout(batch, set.columns, D, g->dtype == SD_F32 && !g->kv_bits, set.stage_bytes);
    s->lay = TileLayout{lay.stages, 0, 0, lay.prefix_off, lay.bar_off, lay.bytes};
    s->q_off = lay.q_off;
    s->buf_off = lay.buf_off;
    s->tile = set.tile;
    s->columns = set.columns;
    s->seg_units = kSegmentUnits;
  }
  if (s->lay.stages < (s->tiles ? kTreeTileLeast : 1) || (s->tiles && g->kv_bits && s->lay.raw_stages < 2))
    return fail(SD_ERR_SHAPE, "batch %d leaves no shared memory for the tiles", batch);
  // a sequence's last pair may be almost empty; no more pairs than columns
  s->pairs = g->n_kv_heads * std::min(int64_t(n_rows) * G, int64_t(n_rows) * G / s->columns + batch);
  s->part_floats = paged_part_floats(s->columns, D);
  s->line_bytes = (int64_t(2) * (batch + 1) * 4 + 127) / 128 * 128;
  const int64_t all = int64_t(n_rows) * n_q_heads;
  s->node_bytes = s->tiles ? 0 : (all * 8 + 127) / 128 * 128 + all * D * 4;
  s->bytes = s->line_bytes + (s->pairs + s->ctas) * s->part_floats * 4 + s->node_bytes;
  if (s->pairs + s->ctas >= (int64_t(1) << 30)) return fail(SD_ERR_SHAPE, "too many rows at once (%d)", n_rows);
  return SD_OK;
}

int32_t check_tree(const sd_pages* g, int32_t batch, int32_t n_rows, int32_t n_q_heads) {
  if (int32_t rc = check_pages(g)) return rc;
  if (batch < 0 || batch > kPagedMaxBatch) return fail(SD_ERR_SHAPE, "batch must be in [0, %d] (got %d)", kPagedMaxBatch, batch);
  if (n_rows < 0) return fail(SD_ERR_INVALID_ARG, "n_rows must not be negative");
  if (n_q_heads < 1 || n_q_heads % g->n_kv_heads)
    return fail(SD_ERR_SHAPE, "n_q_heads (%d) is not a positive multiple of n_kv_heads (%d)", n_q_heads, g->n_kv_heads);
  if (n_q_heads > 65536) return fail(SD_ERR_SHAPE, "too many heads");
  if (n_q_heads / g->n_kv_heads > 16)
    return fail(SD_ERR_SHAPE, "at most 16 query heads per kv head (got %d)", n_q_heads / g->n_kv_heads);
  return SD_OK;
}

}  // namespace

extern "C" {

int32_t sd_paged_plan(const sd_plan* g, int32_t* device_flags, sd_stream stream) {
  if (!g) return fail(SD_ERR_INVALID_ARG, "plan is NULL");
  if (g->batch < 0 || g->batch > kPagedMaxBatch)
    return fail(SD_ERR_SHAPE, "batch must be in [0, %d] (got %d)", kPagedMaxBatch, g->batch);
  if (g->table_width < 0 || g->n_rows < 0 || g->n_free < 0 || g->nodes < 0 || g->parents_stride < 0)
    return fail(SD_ERR_INVALID_ARG, "table_width, n_rows, n_free, nodes and parents_stride must not be negative");
  if (!good_page(g->page_size)) return fail(SD_ERR_SHAPE, "page_size must be 16, 32, 64, 128 or 256 (got %d)", g->page_size);
  // a thread's rows and its steps over them are counted in 32 bits
  if (g->n_rows >= (1 << 30)) return fail(SD_ERR_SHAPE, "a plan has fewer than 2^30 rows (got %d)", g->n_rows);
  if (int64_t(g->table_width) * g->page_size >= (int64_t(1) << 31) - 512)
    return fail(SD_ERR_SHAPE, "table_width * page_size tokens must stay below 2^31");
  if (g->batch && (!g->lengths || !g->added || (g->table_width && !g->tables) || !g->ends))
    return fail(SD_ERR_INVALID_ARG, "NULL argument");
  if (!g->first || (g->n_rows && (!g->seq || !g->positions))) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  const bool grow = g->held || g->free_pages || g->taken;
  if (grow && (!g->held || !g->taken || (g->n_free && !g->free_pages)))
    return fail(SD_ERR_INVALID_ARG, "held, free_pages and taken come together");
  if (g->parents && (g->nodes < 1 || g->nodes > SD_MAX_NODES))
    return fail(SD_ERR_SHAPE, "a tree has 1 to %d nodes (got %d)", SD_MAX_NODES, g->nodes);
  if (any_misaligned4({g->lengths, g->added, g->tables, g->held, g->free_pages, g->taken, g->parents, g->first, g->ends, g->seq,
                       g->positions, g->places, device_flags}) || misaligned(g->slots, 8) || misaligned(g->masks, 8))
    return fail(SD_ERR_INVALID_ARG, "an array is misaligned");
  // every block reads the inputs, and some after another has written
  const int64_t B = g->batch, N = g->n_rows;
  const std::pair<const void*, int64_t> in[] = {
      {g->lengths, 4 * B}, {g->added, 4 * B}, {g->tables, 4 * B * g->table_width}, {g->held, 4 * B},
      {g->free_pages, 4 * int64_t(g->n_free)}, {g->taken, 4},
      {g->parents, g->parents && B ? 4 * ((B - 1) * g->parents_stride + g->nodes) : 0}};
  const std::pair<const void*, int64_t> to[] = {
      {g->first, 4 * (B + 1)}, {g->ends, 4 * B}, {g->seq, 4 * N}, {g->positions, 4 * N}, {g->slots, 8 * N}, {g->places, 4 * N}, {g->masks, 8 * N}};
  for (const auto& o : to)
    for (const auto& i : in)
      if (o.first && i.first && static_cast<const char*>(o.first) < static_cast<const char*>(i.first) + i.second &&
          static_cast<const char*>(i.first) < static_cast<const char*>(o.first) + o.second)
        return fail(SD_ERR_INVALID_ARG, "an output lies in one of the inputs");
  int sms = 0;
  if (int32_t rc = sm_count(&sms)) return rc;
  PlanParams p{};
  p.lengths = g->lengths;
  p.added = g->added;
  p.tables = g->tables;
  p.held = g->held;
  p.free_pages = g->free_pages;
  p.taken = g->taken;
  p.parents = g->parents;
  p.parents_stride = g->parents_stride;
  p.n_free = g->n_free;
  p.T = g->nodes;
  p.B = g->batch;
  p.W = g->table_width;
  p.P = g->page_size;
  p.page_shift = log2_of(g->page_size);
  p.N = g->n_rows;
  p.first = g->first;
  p.ends = g->ends;
  p.seq = g->seq;
  p.positions = g->positions;
  p.places = g->places;
  p.slots = g->slots;
  p.masks = g->masks;
  p.flags = device_flags;
  // a thread per few rows, or a warp per tree
  const int64_t threads = g->parents ? int64_t(g->batch) * 32 : (int64_t(g->n_rows) + kPlanRows - 1) / kPlanRows;
  const int grid = int(std::max<int64_t>(1, std::min<int64_t>((threads + kPlanThreads - 1) / kPlanThreads, 2 * sms)));
  const size_t smem = plan_smem(g->batch);
  const void* fn = plan_kernel_ptr();
  if (smem > 48 * 1024) SD_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, plan_smem(kPagedMaxBatch)));
  p.rows = true;
  p.commit = grow && grid <= kPlanCluster;
  void* args[1] = {&p};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int32_t rc = launch(fn, dim3(unsigned(grid)), kPlanThreads, smem, st, args, p.commit ? grid : 1)) return rc;
  if (grow && !p.commit) {
    p.rows = false;
    p.commit = true;
    return launch(fn, dim3(kPlanCluster), kPlanThreads, smem, st, args, kPlanCluster);
  }
  return SD_OK;
}

int32_t sd_paged_tree_workspace(const sd_pages* g, int32_t batch, int32_t n_rows, int32_t n_q_heads, int64_t* bytes) {
  if (!bytes) return fail(SD_ERR_INVALID_ARG, "bytes is NULL");
  *bytes = 0;
  if (int32_t rc = check_tree(g, batch, n_rows, n_q_heads)) return rc;
  if (batch == 0 || n_rows == 0) return SD_OK;
  TreeShape s{};
  if (int32_t rc = tree_shape(g, batch, n_rows, n_q_heads, &s)) return rc;
  *bytes = s.bytes;
  return SD_OK;
}

int32_t sd_paged_tree_decode(const sd_pages* g, int32_t layer, const void* q, int32_t n_rows, int32_t batch,
                             int32_t n_q_heads, const int32_t* tables, int32_t table_width, const int32_t* lengths,
                             const int32_t* first, const int64_t* masks, const int32_t* places, float scale,
                             int32_t window, const float* sinks, void* out, void* workspace, int64_t workspace_bytes,
                             int32_t* device_flags, sd_stream stream) {
  if (int32_t rc = check_tree(g, batch, n_rows, n_q_heads)) return rc;
  if (int32_t rc = check_layer(g, layer)) return rc;
  if (batch == 0 || n_rows == 0) return SD_OK;
  if (!q || !tables || !lengths || !first || !out || !workspace) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  if (!std::isfinite(scale)) return fail(SD_ERR_INVALID_ARG, "scale must be finite");
  if (window < 0) return fail(SD_ERR_INVALID_ARG, "window must not be negative");
  if (table_width < 1) return fail(SD_ERR_INVALID_ARG, "table_width must be positive");
  if (int64_t(table_width) * g->page_size >= (int64_t(1) << 31) - 512)
    return fail(SD_ERR_SHAPE, "table_width * page_size tokens must stay below 2^31");
  if (misaligned(q, 16) || misaligned(out, 16) || misaligned(workspace, 16))
    return fail(SD_ERR_INVALID_ARG, "q, out and workspace must be 16-byte aligned");
  if (any_misaligned4({tables, lengths, first, places, sinks, device_flags}) || misaligned(masks, 8))
    return fail(SD_ERR_INVALID_ARG, "an array is misaligned");
  TreeShape s{};
  if (int32_t rc = tree_shape(g, batch, n_rows, n_q_heads, &s)) return rc;
  if (workspace_bytes < s.bytes)
    return fail(SD_ERR_CAPACITY, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)s.bytes);
  const int D = g->head_dim, G = n_q_heads / g->n_kv_heads;
  const int64_t max_tiles = (int64_t(table_width) * g->page_size + s.tile - 1) / s.tile + s.seg_units;
  if (max_tiles * s.pairs >= (int64_t(1) << 31)) return fail(SD_ERR_SHAPE, "rows * table_width too large");
  const int64_t columns = int64_t(n_rows) * G, blocks = (columns + kTreeMergeCols - 1) / kTreeMergeCols * g->n_kv_heads;
  if (columns >= (int64_t(1) << 31) - kTreeMergeCols || blocks >= (int64_t(1) << 31))
    return fail(SD_ERR_SHAPE, "too many rows at once (%d)", n_rows);

  const int64_t rows = layer_rows(g) * layer;
  const int rb = row_bytes(g), box = std::min(g->page_size, s.tile);
  TreeParams p{};
  p.k_data = static_cast<uint8_t*>(at(g->k_data, rows * rb));
  p.v_data = static_cast<uint8_t*>(at(g->v_data, rows * rb));
  CUtensorMap tmK, tmV;
  if (int32_t rc = encode_map(&tmK, const_cast<uint8_t*>(p.k_data), rb, layer_rows(g), box, !s.tiles, !s.tiles || !g->kv_bits)) return rc;
  if (int32_t rc = encode_map(&tmV, const_cast<uint8_t*>(p.v_data), rb, layer_rows(g), box, !s.tiles, !s.tiles || !g->kv_bits)) return rc;
  p.q = q;
  p.out = out;
  p.line = static_cast<int*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + s.line_bytes);
  if (s.node_bytes) {
    p.node_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + s.bytes - s.node_bytes);
    p.node_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + s.bytes - int64_t(n_rows) * n_q_heads * D * 4);
  }
  p.by_g.set(G);
  p.tables = tables;
  p.lengths = lengths;
  p.first = first;
  p.masks = masks;
  p.places = places;
  p.sinks = sinks;
  if (g->kv_bits) {
    const int64_t off = rows * sb_bytes(g);
    p.k_scales = at(g->k_scales, off);
    p.k_biases = at(g->k_biases, off);
    p.v_scales = at(g->v_scales, off);
    p.v_biases = at(g->v_biases, off);
  }
  p.n_pages = g->n_pages;
  p.B = batch;
  p.Hkv = g->n_kv_heads;
  p.Hq = n_q_heads;
  p.G = G;
  p.P = g->page_size;
  p.W = table_width;
  p.N = n_rows;
  p.window = window;
  p.RT = s.columns;
  p.seg_units = s.seg_units;
  p.part_floats = s.part_floats;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.magic = 0x64006400u;
  p.flags = device_flags;
  p.stages = s.lay.stages;
  p.raw_stages = s.lay.raw_stages;
  p.q_off = s.q_off;
  p.buf_off = s.buf_off;
  p.prefix_off = s.lay.prefix_off;
  p.bar_off = s.lay.bar_off;
  p.ncta = s.ctas;
  SD_CUDA(cudaFuncSetAttribute(s.attend, cudaFuncAttributeMaxDynamicSharedMemorySize, s.smem_most));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* args[3] = {&p, &tmK, &tmV};
  if (int32_t rc = launch(s.attend, dim3(unsigned(p.ncta)), s.threads, size_t(s.lay.bytes), st, args)) return rc;
  return launch(s.merge, dim3(unsigned(blocks)), kTreeMergeCols * D / 4, 0, st, args);
}

int32_t sd_paged_keep(const sd_pages* g, const int32_t* tables, int32_t batch, int32_t table_width,
                      const int32_t* ends, const int32_t* first, const int32_t* path, int32_t path_width,
                      const int32_t* kept, int32_t* new_lengths, int32_t* device_flags, sd_stream stream) {
  if (int32_t rc = check_pages(g)) return rc;
  if (batch < 0 || batch > kPagedMaxBatch) return fail(SD_ERR_SHAPE, "batch must be in [0, %d] (got %d)", kPagedMaxBatch, batch);
  if (path_width < 0 || path_width > SD_MAX_NODES)
    return fail(SD_ERR_SHAPE, "path_width must be in [0, %d] (got %d)", SD_MAX_NODES, path_width);
  if (batch == 0) return SD_OK;
  if (!tables || !ends || !first || (path_width && !path) || !kept || !new_lengths) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  if (table_width < 1) return fail(SD_ERR_INVALID_ARG, "table_width must be positive");
  if (int64_t(table_width) * g->page_size >= (int64_t(1) << 31) - 512)
    return fail(SD_ERR_SHAPE, "table_width * page_size tokens must stay below 2^31");
  if (any_misaligned4({tables, ends, first, path, kept, new_lengths, device_flags}))
    return fail(SD_ERR_INVALID_ARG, "an int32 array is misaligned");
  // every block reads ends, first and kept of its sequence, and some after another has written the new length
  const int32_t *n0 = new_lengths, *n1 = new_lengths + batch;
  auto meets = [&](const int32_t* a, int64_t n) { return a < n1 && n0 < a + n; };
  if (meets(ends, batch) || meets(first, batch + 1) || meets(kept, batch) || meets(path, int64_t(batch) * path_width) ||
      meets(tables, int64_t(batch) * table_width))
    return fail(SD_ERR_INVALID_ARG, "new_lengths must be none of the inputs");
  KeepParams p{};
  p.tables = tables;
  p.ends = ends;
  p.first = first;
  p.path = path;
  p.kept = kept;
  p.lengths = new_lengths;
  p.B = batch;
  p.W = table_width;
  p.P = g->page_size;
  p.page_shift = log2_of(g->page_size);
  p.T = path_width;
  p.Hkv = g->n_kv_heads;
  p.n_pages = g->n_pages;
  p.flags = device_flags;
  void* a[6] = {g->k_data, g->v_data, g->k_scales, g->k_biases, g->v_scales, g->v_biases};
  for (int i = 0; i < (g->kv_bits ? 6 : 2); ++i) {
    p.array[i] = static_cast<uint8_t*>(a[i]);
    p.row[i] = i < 2 ? row_bytes(g) : sb_bytes(g);
    p.layer[i] = layer_rows(g) * p.row[i];
    const int64_t columns = int64_t(g->n_kv_heads) * (p.row[i] / std::min(p.row[i], 16));
    if (columns + p.all_columns >= (int64_t(1) << 31)) return fail(SD_ERR_SHAPE, "too many heads");
    p.columns[i] = int(columns);
    p.all_columns += int(columns);
  }
  const int64_t blocks = int64_t(batch) * g->n_layers;
  if (blocks >= (int64_t(1) << 31)) return fail(SD_ERR_SHAPE, "batch * n_layers too large");
  void* args[1] = {&p};
  return launch(keep_kernel_ptr(), dim3(unsigned(blocks)), kKeepThreads, 0, static_cast<cudaStream_t>(stream), args);
}

}  // extern "C"
