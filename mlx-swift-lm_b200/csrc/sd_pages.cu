// sd_pages.cu -- the C ABI of the paged serving cache: argument checks,
// launch shapes and launches (kernels in sd_paged.cuh and sd_rotary.cu) and
// the host-side page map. Host code only.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <unordered_map>
#include <vector>

#include "sd_paged.h"
#include "sd_pages_host.h"

namespace {

using namespace sd;

sd::PagedSet lookup(int dtype, int bits, int D, int G) {
  switch (dtype * 16 + bits) {
    case 0 * 16 + 0: return sd::paged_e0_b0(D, G);
    case 1 * 16 + 0: return sd::paged_e1_b0(D, G);
    case 2 * 16 + 0: return sd::paged_e2_b0(D, G);
    case 0 * 16 + 4: return sd::paged_e0_b4(D, G);
    case 1 * 16 + 4: return sd::paged_e1_b4(D, G);
    case 2 * 16 + 4: return sd::paged_e2_b4(D, G);
    case 0 * 16 + 8: return sd::paged_e0_b8(D, G);
    case 1 * 16 + 8: return sd::paged_e1_b8(D, G);
    case 2 * 16 + 8: return sd::paged_e2_b8(D, G);
    default: return sd::PagedSet{nullptr, nullptr, 0, 0};
  }
}

// CTAs of a decode launch: two per SM, all resident.
int decode_ctas(int sms) { return 2 * sms; }

int32_t check_rows(const sd_rows* r, int32_t heads, int dtype, const char* name) {
  if (heads == 0) return SD_OK;
  if (!r || !r->data) return fail(SD_ERR_INVALID_ARG, "%s is NULL", name);
  if (misaligned(r->data, elt_size(dtype))) return fail(SD_ERR_INVALID_ARG, "%s is misaligned", name);
  return SD_OK;
}

int32_t check_rotation(const sd_rotation* rot, int32_t head_dim, int dtype) {
  if (rot->rot_dim < 0 || rot->rot_dim > head_dim || rot->rot_dim % 2)
    return fail(SD_ERR_SHAPE, "rot_dim must be even and in [0, %d] (got %d)", head_dim, rot->rot_dim);
  if (rot->rot_dim && !rot->inv_freq) return fail(SD_ERR_INVALID_ARG, "inv_freq is NULL");
  if (misaligned(rot->inv_freq, 4) || misaligned(rot->q_norm, elt_size(dtype)) || misaligned(rot->k_norm, elt_size(dtype)))
    return fail(SD_ERR_INVALID_ARG, "inv_freq or a norm is misaligned");
  if (!std::isfinite(rot->factor) || !(rot->eps >= 0.0f) || !std::isfinite(rot->eps))
    return fail(SD_ERR_INVALID_ARG, "factor must be finite, eps finite and not negative");
  if (rot->reserved[0] || rot->reserved[1]) return fail(SD_ERR_INVALID_ARG, "reserved fields must be 0");
  return SD_OK;
}

sd::Rows rows_of(const sd_rows* r) {
  return r ? sd::Rows{r->data, r->batch_stride, r->token_stride, r->head_stride} : sd::Rows{};
}

// Largest access, in elements, that every row start and chunk of these rows allows.
void limit_vec(const sd::Rows& r, int heads, int esize, int* vec) {
  if (heads == 0) return;
  while (*vec > 1 && (misaligned(r.data, size_t(*vec) * esize) || r.batch % *vec || r.token % *vec || r.head % *vec)) *vec /= 2;
}

int32_t launch_rotary(sd::RotaryParams& p, int64_t n_tokens, bool traditional, int dtype, int bits, cudaStream_t st) {
  // a warp's last group of tokens may reach 31 past the end, in 32-bit indexes
  if (n_tokens >= (int64_t(1) << 31) - 64)
    return fail(SD_ERR_SHAPE, "a call takes fewer than 2^31 - 64 tokens (got %lld)", (long long)n_tokens);
  const int es = elt_size(dtype);
  int vec = 16 / es;
  limit_vec(p.q, p.Hq, es, &vec);
  limit_vec(p.q_out, p.Hq, es, &vec);
  limit_vec(p.k, p.Hkv, es, &vec);
  limit_vec(p.v, p.Hv, es, &vec);
  if (!p.tables) limit_vec(p.k_out, p.Hkv, es, &vec);
  while (vec > 1 && p.D % (2 * vec)) vec /= 2;  // chunk pairs must tile the head
  // In the half layout each rotated half must be whole chunks too, down to two
  // elements; with an odd number of rotations the kernel fetches the other
  // elements one by one from shared memory instead, four to a chunk (6023
  // tokens of 48 heads of 128 in bf16: 61 rotations 61 us so, 107 with
  // one-element chunks; 62 and 60 rotations 62 and 62 us so, 57 and 40 with
  // chunks of two and four).
  int even = vec;
  while (even > 1 && p.rot2 % even) even /= 2;
  const bool shifted = !traditional && vec >= 4 && even == 1 && p.rot2 > 0;
  if (!traditional) vec = shifted ? 4 : even;
  // Quantizing makes a small call wait for a lane's divisions: half the
  // elements per lane then, 16 users' appends to an 8-bit pool 4.7 -> 3.9 us.
  const int64_t rows = n_tokens * (p.Hq + p.Hkv + p.Hv);
  if (bits && rows < 4 * sd::kRotFill) vec = std::min(vec, 4);
  const int lg_log = sd::rotary_lanes_log(p.D, vec), groups = 32 >> lg_log, warps = sd::kRotThreads / 32;
  // A warp's groups of lanes each take one row per pass. The more passes a
  // warp makes, the more rows share its cos, sin and weights; the fewer, the
  // more warps there are. So: as many as leave about kRotFill warps, at most
  // kRotPasses, over more than one token where the heads are few.
  const int heads[3] = {p.Hq, p.Hkv, p.Hv};
  const int64_t passes = rows / groups;
  const int span = int(std::min<int64_t>(sd::kRotPasses, std::max<int64_t>(1, passes / sd::kRotFill)));
  int64_t units = 0;
  for (int i = 0; i < 3; ++i) {
    sd::RotaryParams::Kind& k = p.kind[i];
    k.first = int(units);
    k.tok_log = 0;
    while ((2 << k.tok_log) <= groups && heads[i] * (2 << k.tok_log) <= span * groups) ++k.tok_log;
    const int step = groups >> k.tok_log, per = ((heads[i] + step - 1) / step + span - 1) / span;
    k.span = span;
    k.per.set(std::max(per, 1));
    units += ((n_tokens + (1 << k.tok_log) - 1) >> k.tok_log) * per;
    if (units >= (int64_t(1) << 31) - warps - 64)
      return fail(SD_ERR_SHAPE, "too many rows at once (%lld tokens)", (long long)n_tokens);
  }
  p.units = int(units);
  p.n_tokens = int(n_tokens);
  p.pairs.set(std::max(p.rot2, 1));
  p.inv_dim = 1.0f / float(p.D);
  p.ring_at = (warps * groups * (2 * sd::rotary_pitch(p.rot2) * 4 + (bits ? p.D * es : 0)) + 15) / 16 * 16;
  const bool wide = p.D > 128;
  const int pass = 32 * (vec >= 4 ? 1 : (wide ? 2 : 1) * (2 / vec)) * 2 * vec * es;
  const size_t smem = size_t(p.ring_at) + size_t(warps) * sd::kRotDepth * pass;
  const void* fn = sd::rotary_kernel_for(dtype, bits, vec, wide, shifted, traditional);
  void* args[1] = {&p};
  return launch(fn, dim3(unsigned((p.units + warps - 1) / warps)), sd::kRotThreads, smem, st, args);
}

void set_rotation(sd::RotaryParams& p, const sd_rotation* rot) {
  p.inv_freq = rot->inv_freq;
  p.q_norm = rot->q_norm;
  p.k_norm = rot->k_norm;
  p.eps = rot->eps;
  p.factor = rot->factor;
  p.rot2 = rot->rot_dim / 2;
}

}  // namespace

extern "C" {

int32_t sd_rotary(const sd_rotation* rot, int32_t dtype, int32_t head_dim, int32_t batch, int32_t tokens,
                  const int32_t* positions, int32_t n_q_heads, const sd_rows* q, const sd_rows* q_out,
                  int32_t n_kv_heads, const sd_rows* k, const sd_rows* k_out, sd_stream stream) {
  if (!rot) return fail(SD_ERR_INVALID_ARG, "rot is NULL");
  if (int32_t rc = check_dtype(dtype)) return rc;
  if (head_dim < 2 || head_dim > 256 || head_dim % 2)
    return fail(SD_ERR_SHAPE, "head_dim must be even and in [2, 256] (got %d)", head_dim);
  if (batch < 0 || tokens < 0 || n_q_heads < 0 || n_kv_heads < 0)
    return fail(SD_ERR_INVALID_ARG, "batch, tokens and head counts must not be negative");
  if (int32_t rc = check_rotation(rot, head_dim, dtype)) return rc;
  if (batch == 0 || tokens == 0 || (n_q_heads == 0 && n_kv_heads == 0)) return SD_OK;
  if (!positions || misaligned(positions, 4)) return fail(SD_ERR_INVALID_ARG, "positions is NULL or misaligned");
  for (int32_t rc : {check_rows(q, n_q_heads, dtype, "q"), check_rows(q_out, n_q_heads, dtype, "q_out"),
                     check_rows(k, n_kv_heads, dtype, "k"), check_rows(k_out, n_kv_heads, dtype, "k_out")})
    if (rc != SD_OK) return rc;
  if (int64_t(n_q_heads) + n_kv_heads > 65536) return fail(SD_ERR_SHAPE, "too many heads");
  sd::RotaryParams p{};
  p.q = rows_of(q);
  p.q_out = rows_of(q_out);
  p.k = rows_of(k);
  p.k_out = rows_of(k_out);
  p.Hq = n_q_heads;
  p.Hkv = n_kv_heads;
  p.D = head_dim;
  p.L.set(tokens);
  p.positions = positions;
  set_rotation(p, rot);
  return launch_rotary(p, int64_t(batch) * tokens, rot->traditional != 0, dtype, 0, static_cast<cudaStream_t>(stream));
}

int32_t sd_paged_append(const sd_pages* g, int32_t layer, int32_t n_tokens, const sd_rows* k, const sd_rows* v,
                        const int32_t* tables, int32_t batch, int32_t table_width, const int32_t* positions,
                        const int32_t* seq, const sd_rotation* rot, int32_t n_q_heads, const sd_rows* q,
                        const sd_rows* q_out, int32_t* device_flags, sd_stream stream) {
  if (int32_t rc = check_pages(g)) return rc;
  if (int32_t rc = check_layer(g, layer)) return rc;
  if (n_tokens < 0 || batch < 0 || table_width < 0 || n_q_heads < 0)
    return fail(SD_ERR_INVALID_ARG, "n_tokens, batch, table_width and n_q_heads must not be negative");
  if (n_q_heads > 0 && !rot) return fail(SD_ERR_INVALID_ARG, "queries are only taken along with a rotation");
  if (rot)
    if (int32_t rc = check_rotation(rot, g->head_dim, g->dtype)) return rc;
  if (n_tokens == 0) return SD_OK;
  if (!tables || !positions) return fail(SD_ERR_INVALID_ARG, "tables or positions is NULL");
  if (misaligned(tables, 4) || misaligned(positions, 4) || misaligned(seq, 4) || misaligned(device_flags, 4))
    return fail(SD_ERR_INVALID_ARG, "an int32 array is misaligned");
  for (int32_t rc : {check_rows(k, g->n_kv_heads, g->dtype, "k"), check_rows(v, g->n_kv_heads, g->dtype, "v"),
                     check_rows(q, n_q_heads, g->dtype, "q"), check_rows(q_out, n_q_heads, g->dtype, "q_out")})
    if (rc != SD_OK) return rc;
  if (int64_t(n_q_heads) + 2 * int64_t(g->n_kv_heads) > 65536) return fail(SD_ERR_SHAPE, "too many heads");
  sd::RotaryParams p{};
  p.q = rows_of(n_q_heads ? q : nullptr);
  p.q_out = rows_of(n_q_heads ? q_out : nullptr);
  p.k = rows_of(k);
  p.v = rows_of(v);
  p.Hq = n_q_heads;
  p.Hkv = p.Hv = g->n_kv_heads;
  p.D = g->head_dim;
  p.L.set(n_tokens);
  p.positions = positions;
  if (rot) set_rotation(p, rot);
  p.tables = tables;
  p.seq = seq;
  p.B = batch;
  p.W = table_width;
  p.P = g->page_size;
  p.page_shift = log2_of(g->page_size);
  p.n_pages = g->n_pages;
  const int64_t rows = layer_rows(g) * layer;
  p.k_data = at(g->k_data, rows * row_bytes(g));
  p.v_data = at(g->v_data, rows * row_bytes(g));
  if (g->kv_bits) {
    p.k_scales = at(g->k_scales, rows * sb_bytes(g));
    p.k_biases = at(g->k_biases, rows * sb_bytes(g));
    p.v_scales = at(g->v_scales, rows * sb_bytes(g));
    p.v_biases = at(g->v_biases, rows * sb_bytes(g));
  }
  p.flags = device_flags;
  return launch_rotary(p, n_tokens, rot && rot->traditional, g->dtype, g->kv_bits, static_cast<cudaStream_t>(stream));
}

int32_t sd_copy_pages(const sd_pages* g, const int32_t* src, const int32_t* dst, int32_t n, int32_t* device_flags,
                      sd_stream stream) {
  if (int32_t rc = check_pages(g)) return rc;
  if (n < 0) return fail(SD_ERR_INVALID_ARG, "n must not be negative");
  if (n == 0) return SD_OK;
  if (!src || !dst) return fail(SD_ERR_INVALID_ARG, "src or dst is NULL");
  if (misaligned(src, 4) || misaligned(dst, 4) || misaligned(device_flags, 4))
    return fail(SD_ERR_INVALID_ARG, "an int32 array is misaligned");
  sd::CopyParams p{};
  p.src = src;
  p.dst = dst;
  p.n = n;
  p.n_pages = g->n_pages;
  void* a[6] = {g->k_data, g->v_data, g->k_scales, g->k_biases, g->v_scales, g->v_biases};
  for (int i = 0; i < (g->kv_bits ? 6 : 2); ++i) {
    p.array[i] = static_cast<uint8_t*>(a[i]);
    p.bytes[i] = int64_t(g->n_kv_heads) * g->page_size * (i < 2 ? row_bytes(g) : sb_bytes(g));
    p.pieces[i] = int((p.bytes[i] + sd::kCopyPiece - 1) / sd::kCopyPiece);
    p.per_pair += p.pieces[i];
  }
  p.flags = device_flags;
  const int64_t pieces = int64_t(n) * g->n_layers * p.per_pair;
  if (pieces >= (int64_t(1) << 31)) return fail(SD_ERR_SHAPE, "too many pages at once (%d)", n);
  void* args[1] = {&p};
  return launch(sd::copy_pages_kernel_ptr(), dim3(unsigned(pieces)),
                sd::kCopyThreads, 0, static_cast<cudaStream_t>(stream), args);
}

// two segments (o, m, l) per CTA
static int64_t workspace_bytes_of(const sd_pages* g, int32_t n_q_heads, int ctas) {
  return int64_t(ctas) * 2 * sd::paged_part_floats(n_q_heads / g->n_kv_heads, g->head_dim) * 4;
}

static int32_t check_heads(const sd_pages* g, int32_t batch, int32_t n_q_heads) {
  if (batch < 1 || batch > sd::kPagedMaxBatch) return fail(SD_ERR_SHAPE, "batch must be in [1, %d] (got %d)", sd::kPagedMaxBatch, batch);
  if (n_q_heads < 1 || n_q_heads % g->n_kv_heads)
    return fail(SD_ERR_SHAPE, "n_q_heads (%d) is not a positive multiple of n_kv_heads (%d)", n_q_heads, g->n_kv_heads);
  if (n_q_heads > 65536) return fail(SD_ERR_SHAPE, "too many heads");  // the kernels index head * D in 32 bits
  if (n_q_heads / g->n_kv_heads > 16) return fail(SD_ERR_SHAPE, "at most 16 query heads per kv head (got %d)", n_q_heads / g->n_kv_heads);
  return SD_OK;
}

int32_t sd_paged_workspace(const sd_pages* g, int32_t batch, int32_t n_q_heads, int64_t* bytes) {
  if (!bytes) return fail(SD_ERR_INVALID_ARG, "bytes is NULL");
  *bytes = 0;
  if (int32_t rc = check_pages(g)) return rc;
  if (int32_t rc = check_heads(g, batch, n_q_heads)) return rc;
  int sms = 0;
  if (int32_t rc = sm_count(&sms)) return rc;
  *bytes = workspace_bytes_of(g, n_q_heads, decode_ctas(sms));
  return SD_OK;
}

int32_t sd_paged_decode(const sd_pages* g, int32_t layer, const void* q, int32_t batch, int32_t n_q_heads,
                        const int32_t* tables, int32_t table_width, const int32_t* lengths, float scale,
                        int32_t window, const float* sinks, void* out, void* workspace, int64_t workspace_bytes,
                        int32_t* device_flags, sd_stream stream) {
  if (int32_t rc = check_pages(g)) return rc;
  if (int32_t rc = check_layer(g, layer)) return rc;
  if (batch == 0) return SD_OK;
  if (int32_t rc = check_heads(g, batch, n_q_heads)) return rc;
  if (!q || !tables || !lengths || !out || !workspace) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  if (!std::isfinite(scale)) return fail(SD_ERR_INVALID_ARG, "scale must be finite");
  if (window < 0) return fail(SD_ERR_INVALID_ARG, "window must not be negative");
  if (table_width < 1) return fail(SD_ERR_INVALID_ARG, "table_width must be positive");
  if (int64_t(table_width) * g->page_size >= (int64_t(1) << 31) - 512)
    return fail(SD_ERR_SHAPE, "table_width * page_size tokens must stay below 2^31");
  if (misaligned(q, 16) || misaligned(out, 16) || misaligned(workspace, 16))
    return fail(SD_ERR_INVALID_ARG, "q, out and workspace must be 16-byte aligned");
  if (misaligned(tables, 4) || misaligned(lengths, 4) || misaligned(sinks, 4) || misaligned(device_flags, 4))
    return fail(SD_ERR_INVALID_ARG, "an int32 or fp32 array is misaligned");
  const int D = g->head_dim, G = n_q_heads / g->n_kv_heads;
  const sd::PagedSet ks = lookup(g->dtype, g->kv_bits, D, G);
  if (!ks.decode) return fail(SD_ERR_SHAPE, "no kernel for dtype %d, bits %d, head_dim %d", g->dtype, g->kv_bits, D);
  // most units (tiles and segment ends) of one sequence and kv head
  const int64_t max_tiles = (int64_t(table_width) * g->page_size + ks.tile - 1) / ks.tile + sd::kSegmentUnits;
  if (max_tiles * batch * g->n_kv_heads >= (int64_t(1) << 31)) return fail(SD_ERR_SHAPE, "batch * table_width too large");
  int sms = 0;
  if (int32_t rc = sm_count(&sms)) return rc;
  const int max_ctas = decode_ctas(sms);
  if (workspace_bytes < workspace_bytes_of(g, n_q_heads, max_ctas))
    return fail(SD_ERR_CAPACITY, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)workspace_bytes_of(g, n_q_heads, max_ctas));

  const int64_t rows = layer_rows(g);
  const int rb = row_bytes(g), box = std::min(g->page_size, ks.tile);
  CUtensorMap tmK, tmV;
  if (int32_t rc = sd::encode_map(&tmK, at(g->k_data, rows * layer * rb), rb, rows, box)) return rc;
  if (int32_t rc = sd::encode_map(&tmV, at(g->v_data, rows * layer * rb), rb, rows, box)) return rc;

  sd::PagedParams p{};
  p.q = q;
  p.out = out;
  p.part = static_cast<float*>(workspace);
  p.tables = tables;
  p.lengths = lengths;
  p.sinks = sinks;
  if (g->kv_bits) {
    const int64_t off = rows * layer * sb_bytes(g);
    p.k_scales = at(g->k_scales, off);
    p.k_biases = at(g->k_biases, off);
    p.v_scales = at(g->v_scales, off);
    p.v_biases = at(g->v_biases, off);
  }
  p.n_pages = g->n_pages;
  p.B = batch;
  p.Hkv = g->n_kv_heads;
  p.G = G;
  p.P = g->page_size;
  p.W = table_width;
  p.window = window;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.magic = 0x64006400u;
  p.flags = device_flags;

  const sd::PagedLayout lay = sd::paged_layout(batch, G, D, g->dtype == SD_F32 && !g->kv_bits, ks.stage_bytes);
  if (lay.stages < 1) return fail(SD_ERR_SHAPE, "batch %d leaves no shared memory for the tiles", batch);
  p.stages = lay.stages;
  p.q_off = lay.q_off;
  p.buf_off = lay.buf_off;
  p.prefix_off = lay.prefix_off;
  p.bar_off = lay.bar_off;
  SD_CUDA(cudaFuncSetAttribute(ks.decode, cudaFuncAttributeMaxDynamicSharedMemorySize, sd::kPagedSmem));

  const int64_t max_units = max_tiles * batch * g->n_kv_heads;
  p.ncta = int(std::min<int64_t>(max_ctas, max_units));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* args[3] = {&p, &tmK, &tmV};
  if (int32_t rc = launch(ks.decode, dim3(unsigned(p.ncta)), sd::kPagedThreads, size_t(lay.bytes), st, args)) return rc;
  void* margs[1] = {&p};
  if (int64_t(batch) * n_q_heads > sd::kMergeMany) {
    const unsigned per = unsigned(n_q_heads + sd::kMergeHeads - 1) / sd::kMergeHeads;
    return launch(ks.merge_many, dim3(unsigned(batch) * per), sd::kMergeThreads, 0, st, margs);
  }
  return launch(ks.merge, dim3(unsigned(batch) * unsigned(n_q_heads)), sd::kMergeThreads, 0, st, margs);
}

}  // extern "C"

// ---------------------------------------------------------------------------
// The page map
// ---------------------------------------------------------------------------

struct sd_pagemap {
  struct Seq {
    std::vector<int32_t> pages;
    int64_t tokens = 0;
  };
  int32_t page_size;
  std::vector<int32_t> refs;       // sequences that hold each page
  std::vector<uint64_t> free_bits; // one bit per free page: the lowest free page is taken first
  int64_t n_free;
  int64_t first_free;              // no free page below this one
  std::unordered_map<int64_t, Seq> seqs;
  int64_t next_id = 0;

  bool is_free(int64_t p) const { return free_bits[p >> 6] >> (p & 63) & 1; }
  int32_t take() {  // n_free > 0
    int64_t w = first_free >> 6;
    while (free_bits[w] == 0) ++w;
    const int64_t p = w * 64 + __builtin_ctzll(free_bits[w]);
    free_bits[w] &= free_bits[w] - 1;
    refs[p] = 1;
    --n_free;
    first_free = p + 1;
    return int32_t(p);
  }
  void drop(int32_t p) {
    if (--refs[p] == 0) {
      free_bits[p >> 6] |= uint64_t(1) << (p & 63);
      ++n_free;
      first_free = std::min<int64_t>(first_free, p);
    }
  }
};

namespace {

template <class F>
int32_t guarded(F f) {  // no exception leaves the C ABI
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(SD_ERR_CAPACITY, "out of host memory");
  } catch (...) {
    return fail(SD_ERR_STATE, "unexpected error in the page map");
  }
}

template <class M>
auto find(M* m, int64_t seq) -> decltype(&m->seqs.begin()->second) {
  auto it = m->seqs.find(seq);
  return it == m->seqs.end() ? nullptr : &it->second;
}

int32_t no_seq(int64_t seq) { return fail(SD_ERR_STATE, "no sequence %lld", (long long)seq); }

}  // namespace

extern "C" {

int32_t sd_pagemap_create(int64_t n_pages, int32_t page_size, sd_pagemap** out) {
  if (!out) return fail(SD_ERR_INVALID_ARG, "out is NULL");
  *out = nullptr;
  if (n_pages < 1 || n_pages >= (int64_t(1) << 31) || page_size < 1)
    return fail(SD_ERR_INVALID_ARG, "n_pages must be in [1, 2^31), page_size positive");
  return guarded([&] {
    sd_pagemap* m = new sd_pagemap();
    try {
      m->page_size = page_size;
      m->refs.assign(size_t(n_pages), 0);
      m->free_bits.assign(size_t((n_pages + 63) / 64), ~uint64_t(0));
      if (n_pages % 64) m->free_bits.back() = (uint64_t(1) << (n_pages % 64)) - 1;
    } catch (...) {
      delete m;
      throw;
    }
    m->n_free = n_pages;
    m->first_free = 0;
    *out = m;
    return int32_t(SD_OK);
  });
}

int32_t sd_pagemap_destroy(sd_pagemap* m) {
  delete m;
  return SD_OK;
}

int32_t sd_pagemap_add(sd_pagemap* m, int64_t* seq) {
  if (!m || !seq) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  return guarded([&] {
    m->seqs.emplace(m->next_id, sd_pagemap::Seq());
    *seq = m->next_id++;
    return int32_t(SD_OK);
  });
}

int32_t sd_pagemap_fork(sd_pagemap* m, int64_t seq, int64_t* forked) {
  if (!m || !forked) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  const sd_pagemap::Seq* s = find(m, seq);
  if (!s) return no_seq(seq);
  return guarded([&] {
    sd_pagemap::Seq copy = *s;
    auto it = m->seqs.emplace(m->next_id, std::move(copy)).first;
    for (int32_t p : it->second.pages) ++m->refs[p];
    *forked = m->next_id++;
    return int32_t(SD_OK);
  });
}

int32_t sd_pagemap_free(sd_pagemap* m, int64_t seq) {
  if (!m) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  auto it = m->seqs.find(seq);
  if (it == m->seqs.end()) return no_seq(seq);
  for (int32_t p : it->second.pages) m->drop(p);
  m->seqs.erase(it);
  return SD_OK;
}

int32_t sd_pagemap_extend(sd_pagemap* m, int64_t seq, int64_t n_tokens, int32_t* src, int32_t* dst,
                          int32_t* n_copies) {
  if (!m || !src || !dst || !n_copies) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  *n_copies = 0;
  if (n_tokens < 0) return fail(SD_ERR_INVALID_ARG, "n_tokens must not be negative");
  sd_pagemap::Seq* s = find(m, seq);
  if (!s) return no_seq(seq);
  if (n_tokens == 0) return SD_OK;
  if (n_tokens >= (int64_t(1) << 31) - s->tokens) return fail(SD_ERR_CAPACITY, "a sequence holds fewer than 2^31 tokens");
  const int64_t tokens = s->tokens + n_tokens, want = (tokens + m->page_size - 1) / m->page_size;
  const int64_t more = want - int64_t(s->pages.size());
  const bool own = s->tokens % m->page_size != 0 && m->refs[s->pages.back()] > 1;  // the page that the new tokens begin in
  if (more + (own ? 1 : 0) > m->n_free)
    return fail(SD_ERR_CAPACITY, "%lld pages needed, %lld free", (long long)(more + (own ? 1 : 0)), (long long)m->n_free);
  return guarded([&] {
    s->pages.reserve(size_t(want));  // the only step that can fail
    if (own) {
      const int32_t old = s->pages.back(), page = m->take();
      m->drop(old);
      s->pages.back() = page;
      *src = old;
      *dst = page;
      *n_copies = 1;
    }
    for (int64_t i = 0; i < more; ++i) s->pages.push_back(m->take());
    s->tokens = tokens;
    return int32_t(SD_OK);
  });
}

int32_t sd_pagemap_trim(sd_pagemap* m, int64_t seq, int64_t n_tokens, int64_t* trimmed) {
  if (!m) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  if (n_tokens < 0) return fail(SD_ERR_INVALID_ARG, "n_tokens must not be negative");
  sd_pagemap::Seq* s = find(m, seq);
  if (!s) return no_seq(seq);
  const int64_t t = std::min(n_tokens, s->tokens);
  s->tokens -= t;
  const size_t keep = size_t((s->tokens + m->page_size - 1) / m->page_size);
  while (s->pages.size() > keep) {
    m->drop(s->pages.back());
    s->pages.pop_back();
  }
  if (trimmed) *trimmed = t;
  return SD_OK;
}

int32_t sd_pagemap_length(const sd_pagemap* m, int64_t seq, int64_t* tokens) {
  if (!m || !tokens) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  const sd_pagemap::Seq* s = find(m, seq);
  if (!s) return no_seq(seq);
  *tokens = s->tokens;
  return SD_OK;
}

int32_t sd_pagemap_width(const sd_pagemap* m, const int64_t* seqs, int32_t n, int32_t* width) {
  if (!m || !width || (n > 0 && !seqs)) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  *width = 1;
  for (int32_t i = 0; i < n; ++i) {
    const sd_pagemap::Seq* s = find(m, seqs[i]);
    if (!s) return no_seq(seqs[i]);
    *width = std::max(*width, int32_t(s->pages.size()));
  }
  return SD_OK;
}

int32_t sd_pagemap_tables(const sd_pagemap* m, const int64_t* seqs, int32_t n, int32_t width, int32_t* tables,
                          int32_t* lengths) {
  if (!m || (n > 0 && (!seqs || !tables))) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  if (width < 1) return fail(SD_ERR_INVALID_ARG, "width must be positive");
  for (int32_t i = 0; i < n; ++i) {
    const sd_pagemap::Seq* s = find(m, seqs[i]);
    if (!s) return no_seq(seqs[i]);
    if (int64_t(s->pages.size()) > width)
      return fail(SD_ERR_SHAPE, "sequence %lld has %zu pages, the table %d columns", (long long)seqs[i], s->pages.size(), width);
  }
  for (int32_t i = 0; i < n; ++i) {
    const sd_pagemap::Seq* s = find(m, seqs[i]);
    int32_t* row = tables + int64_t(i) * width;
    std::copy(s->pages.begin(), s->pages.end(), row);
    std::fill(row + s->pages.size(), row + width, -1);
    if (lengths) lengths[i] = int32_t(s->tokens);
  }
  return SD_OK;
}

int32_t sd_pagemap_free_pages(const sd_pagemap* m, int64_t* n) {
  if (!m || !n) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  *n = m->n_free;
  return SD_OK;
}

int32_t sd_pagemap_compact(sd_pagemap* m, int32_t* src, int32_t* dst, int32_t room, int32_t* n) {
  if (!m || !n || (room > 0 && (!src || !dst))) return fail(SD_ERR_INVALID_ARG, "NULL argument");
  *n = 0;
  if (room < 0) return fail(SD_ERR_INVALID_ARG, "room must not be negative");
  return guarded([&] {
    std::unordered_map<int32_t, int32_t> moved;
    int64_t low = 0, high = int64_t(m->refs.size()) - 1;
    int32_t count = 0;
    // the highest used pages into the lowest free ones: no page is both
    while (count < room) {
      while (low < high && !m->is_free(low)) ++low;
      while (high > low && m->is_free(high)) --high;
      if (low >= high) break;
      src[count] = int32_t(high--);
      dst[count] = int32_t(low++);
      moved.emplace(src[count], dst[count]);
      ++count;
    }
    for (auto& kv : m->seqs)
      for (int32_t& p : kv.second.pages) {
        auto it = moved.find(p);
        if (it != moved.end()) p = it->second;
      }
    for (int32_t i = 0; i < count; ++i) {
      m->refs[dst[i]] = m->refs[src[i]];
      m->refs[src[i]] = 0;
      m->free_bits[dst[i] >> 6] &= ~(uint64_t(1) << (dst[i] & 63));
      m->free_bits[src[i] >> 6] |= uint64_t(1) << (src[i] & 63);
    }
    m->first_free = 0;
    *n = count;
    return int32_t(SD_OK);
  });
}

}  // extern "C"
