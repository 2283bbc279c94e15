// sd_tree.cuh -- attention of the drafted tokens of each sequence, a tree of at
// most 64 nodes, over a paged KV pool.
//
// Sequence b has held = lengths[b] - n tokens before its n nodes, which are rows
// first[b] .. first[b + 1] of q and out. Node i sees the held tokens and the
// nodes j whose bit its mask has; with a window those alone whose place is above
// its own less the window (token t's place is t). For its query head hq,
//   out = sum_t e^(s_t) v_t / (sum_t e^(s_t) + e^(sink)),  s_t = scale q.k_t;
// a row that sees nothing gives zeros.
//
// The held tokens are the same for all nodes (but for the low end of a window),
// the nodes are few and differ from row to row. So the work is in two parts that
// know nothing of each other:
//   * The (node, query head) columns of a kv head are cut into pairs of at most
//     RT columns, and the pairs' tiles of held tokens are one line that CTAs share
//     equally, as in a decode (sd_paged.cuh). Every segment leaves (o, m, l) in
//     the workspace. No mask at all.
//   * The nodes: a warp takes a row and up to four query heads at a time and
//     attends to the visible nodes alone, reading no other node's rows -- what lies
//     there, not-a-numbers included, does not reach it. A CTA has a warp for it,
//     beside the tiles' warps, whose time hides its chain of loads; the others come
//     to its help when they are done (35 sequences of 8 tokens, 31 nodes, 24 query
//     and 3 kv heads in 8-bit codes of an fp16 pool: 120 -> 75 us).
// tree_attend_kernel does both, and tree_merge_kernel joins a column's nodes and
// segments in CTA order. The tile kernel of 16-bit pools and of codes of bf16 ones
// (sd_tree_tile.cu) has the nodes on the line, as a sequence's last tokens.
// Results depend on no timing. Lengths, rows and tables are read on the device
// only, so a captured graph serves growing sequences.
#pragma once

#include "sd_draft.h"
#include "sd_paged.cuh"

namespace sd {

// What one sequence has of a call. A sequence whose numbers cannot be is taken
// for one without tokens, and its rows give zeros. Where first falls anywhere,
// sequences may have rows in common, more in sum than the workspace has room for:
// then none has any (tree_line), and all rows give zeros.
struct TreeSeq {
  int row0, n, held;  // first row, nodes, tokens before them
  int begin, end;     // the tokens on the line: from the first that any node sees, and up to the nodes or with them
  bool bad, falls;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int b) {
  const int f0 = __ldcg(p.first + b), f1 = __ldcg(p.first + b + 1), len = __ldcg(p.lengths + b);
  const int64_t n = int64_t(f1) - f0;
  TreeSeq s;
  s.falls = n < 0;
  s.bad = f0 < 0 || f1 > p.N || n < 0 || n > kMaxNodes || len < n || len > int64_t(p.W) * p.P;
  s.row0 = f0;
  s.n = s.bad ? 0 : int(n);
  s.held = s.n ? len - s.n : 0;
  s.begin = p.window > 0 && s.held >= p.window ? s.held - p.window + 1 : 0;
  s.end = s.held + (p.node_ml ? 0 : s.n);
  return s;
}
// The sequence of row n < first[B]: the last b with first[b] <= n, which has rows.
__device__ __forceinline__ int tree_find(const TreeParams& p, int n) {
  int b = 0, hi = p.B;
  while (hi - b > 1) {
    const int mid = (b + hi) >> 1;
    if (__ldcg(p.first + mid) <= n) b = mid; else hi = mid;
  }
  return b;
}
// The tokens of sequence b on the line, for the producer.
__device__ __forceinline__ TokenRange token_range(const TreeParams& p, int b) {
  const TreeSeq s = tree_seq(p, b);
  return {s.begin, s.end};
}
__device__ __forceinline__ int tree_pairs(const TreeParams& p, const TreeSeq& s) {
  return (s.n * p.G + p.RT - 1) / p.RT * p.Hkv;
}
// Units of one pair on the line: what beginning and ending its segment costs, in tiles, and its tiles.
__device__ __forceinline__ int tree_units(const TreeParams& p, const TreeSeq& s, int tile) {
  return s.end > s.begin ? (s.end + tile - 1) / tile - s.begin / tile + p.seg_units : 0;
}
// The first token that node i sees: `place` is its position.
__device__ __forceinline__ int tree_low(const TreeParams& p, const TreeSeq& s, int node) {
  const int place = p.places ? __ldcg(p.places + s.row0 + node) : s.held + node;
  return p.window > 0 ? max(0, int(min(int64_t(place) + 1 - p.window, int64_t(s.held)))) : 0;
}

// The nodes that node i sees.
__device__ __forceinline__ uint64_t tree_seen(const TreeParams& p, const TreeSeq& s, int node) {
  uint64_t m = p.masks ? uint64_t(__ldcg(reinterpret_cast<const long long*>(p.masks) + s.row0 + node)) : (uint64_t(2) << node) - 1;
  if (s.n < 64) m &= (uint64_t(1) << s.n) - 1;
  if (p.window) {
    const int64_t least = (p.places ? int64_t(__ldcg(p.places + s.row0 + node)) : int64_t(s.held) + node) - p.window;
    if (least >= s.held)  // places are no lower than that
      for (uint64_t left = m; left; left &= left - 1) {
        const int j = __ffsll(left) - 1;
        if ((p.places ? __ldcg(p.places + s.row0 + j) : s.held + j) <= least) m &= ~(uint64_t(1) << j);
      }
  }
  return m;
}

// Units and pairs before each sequence, by all NT threads of the block; tmp: [2 * NT / 32]. No pairs at all: no row has
// anything to see.
template <int NT>
__device__ __forceinline__ void tree_line(const TreeParams& p, int tile, int* units, int* pairs, int* tmp) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (p.B + NT - 1) / NT, b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  int u = 0, k = 0;
  bool bad = false, falls = false;
  for (int b = b0; b < b1; ++b) {
    const TreeSeq s = tree_seq(p, b);
    falls = falls || s.falls;
    const int np = tree_pairs(p, s), nu = tree_units(p, s, tile);
    bad = bad || s.bad;
    units[b + 1] = np * nu;  // of the sequence, for now
    pairs[b + 1] = np;
    k += np;
    u += np * nu;
  }
  if (bad && p.flags && blockIdx.x == 0) atomicOr(p.flags, kErrBadIndex);
  int iu = u, ik = k;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int yu = __shfl_up_sync(0xffffffffu, iu, x), yk = __shfl_up_sync(0xffffffffu, ik, x);
    if (lane >= x) iu += yu, ik += yk;
  }
  if (lane == 31) tmp[2 * warp] = iu, tmp[2 * warp + 1] = ik;
  const bool none = __syncthreads_or(falls);
  u = iu - u, k = ik - k;
  for (int w = 0; w < warp; ++w) u += tmp[2 * w], k += tmp[2 * w + 1];
  if (none) u = k = 0;
  if (tid == 0) units[0] = pairs[0] = 0;
  for (int b = b0; b < b1; ++b) {
    if (!none) u += units[b + 1], k += pairs[b + 1];
    units[b + 1] = u, pairs[b + 1] = k;
    if (blockIdx.x == 0) p.line[b + 1] = u, p.line[p.B + 2 + b] = k;  // for the merge
  }
  if (blockIdx.x == 0 && tid == 0) p.line[0] = p.line[p.B + 1] = 0;
  __syncthreads();
}

struct TreeSegment {
  int b, h, c, pair;   // kv head, which RT columns of it, number of the pair
  int i0, i1;          // tiles
};

// A CTA's way along the line. Pairs of a sequence: kv head by kv head, its columns' pairs side by side, which share
// their tiles in L2.
struct TreeWalk {
  using Seg = TreeSegment;
  const int *units, *pairs;
  int Hkv, seg_units, b, u, u1;
  __device__ __forceinline__ TreeWalk(const TreeParams& p, const int* un, const int* pr, int begin, int end)
      : units(un), pairs(pr), Hkv(p.Hkv), seg_units(p.seg_units), b(0), u(begin), u1(end) {
    int hi = p.B;  // the largest b with units[b] <= u
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (units[mid] <= u) b = mid; else hi = mid;
    }
  }
  __device__ __forceinline__ bool next(TreeSegment& s) {
    while (u < u1) {
      while (units[b + 1] <= u) ++b;  // ends: u < units[B]
      const int np = pairs[b + 1] - pairs[b], nu = (units[b + 1] - units[b]) / np, r = u - units[b], k = r / nu;
      const int per = np / Hkv, first = r - k * nu, last = min(nu, first + u1 - u);
      s.b = b;
      s.h = k / per;
      s.c = k - s.h * per;
      s.pair = pairs[b] + k;
      u += last - first;
      s.i0 = max(first - seg_units, 0);
      s.i1 = last - seg_units;
      if (s.i1 > s.i0) return true;
    }
    return false;
  }
};

// The columns of a pair: x0 + i is (node, query head of the kv head) number x0 + i of the sequence.
struct NodeCols {
  static constexpr bool kLow = true;
  int n, x0, Hq;
  int64_t base, row0;  // of the sequence's first column, of column x0
  FastDiv by_g;
  __device__ __forceinline__ NodeCols(const TreeParams& p, const TreeSeq& s, int h, int c)
      : n(min(p.RT, s.n * p.G - c * p.RT)), x0(c * p.RT), Hq(p.Hq), by_g(p.by_g) {
    base = int64_t(s.row0) * p.Hq + int64_t(h) * p.G;
    row0 = row(0);
  }
  __device__ __forceinline__ int node(int i) const { return by_g(x0 + i); }
  __device__ __forceinline__ int64_t row(int i) const {
    const int nd = node(i);
    return base + int64_t(nd) * Hq + (x0 + i - nd * by_g.d);
  }
};

// Where segment `k` (pair + CTA: both rise along the line, so no two segments share it) lies in the workspace.
__device__ __forceinline__ float* tree_part(const TreeParams& p, int k) { return p.part + int64_t(k) * p.part_floats; }

// ---------------------------------------------------------------------------
// The nodes
// ---------------------------------------------------------------------------

// V neighbouring elements of a row, E each, in fp32.
template <typename E, int V>
__device__ __forceinline__ void load_elements(const E* at, float (&f)[V]) {
  if constexpr (sizeof(E) == 4) {
    if constexpr (V == 4) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(at));
      f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
    } else {
      const float2 x = __ldcg(reinterpret_cast<const float2*>(at));
      f[0] = x.x, f[1] = x.y;
    }
  } else if constexpr (V == 4) {
    const uint2 x = __ldcg(reinterpret_cast<const uint2*>(at));
    unpack_word<E>(x.x, f);
    unpack_word<E>(x.y, f + 2);
  } else {
    unpack_word<E>(__ldcg(reinterpret_cast<const unsigned int*>(at)), f);
  }
}

// One lane's V elements of a stored row, as loaded (the loads of several tokens are under way together) and as values.
template <typename E, int BITS, int V>
struct StoredPiece {
  uint32_t code;
  E scale, bias;
  __device__ __forceinline__ void load(const uint8_t* data, const void* scales, const void* biases, int64_t row, int lane) {
    constexpr int D = 32 * V, ROW = D * BITS / 8, W = V * BITS / 8;
    const uint8_t* at = data + row * ROW + lane * W;
    if constexpr (W == 4) code = __ldcg(reinterpret_cast<const unsigned int*>(at));
    else if constexpr (W == 2) code = __ldcg(reinterpret_cast<const unsigned short*>(at));
    else code = __ldcg(at);
    const int64_t g = row * (D / 64) + lane * V / 64;
    scale = static_cast<const E*>(scales)[g];
    bias = static_cast<const E*>(biases)[g];
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    const float s = Elt<E>::to_f32(scale), b = Elt<E>::to_f32(bias);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = fmaf(float((code >> (BITS * i)) & ((1u << BITS) - 1)), s, b);
  }
};
template <typename E, int V>
struct StoredPiece<E, 0, V> {
  float x[V];
  __device__ __forceinline__ void load(const uint8_t* data, const void*, const void*, int64_t row, int lane) {
    load_elements<E, V>(reinterpret_cast<const E*>(data) + row * (32 * V) + lane * V, x);
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = x[i];
  }
};

// Rows and up to four query heads of one kv head at a time, the CTA's (each grid-th)
// in turn as its warps come for them: `next`, in shared memory, counts, and has the
// number of rows behind it. Which warp has a row changes nothing of it. `any`:
// whether the call has sequences that can be. Lane l holds dimensions [l V, l V + V)
// of q, o and the rows; scores are summed over the lanes by a butterfly that ends
// with head l / 8's in lane l, so that lane l keeps token l % 8's of the eight
// that are taken at a time.
template <typename E, int BITS, int D>
__device__ __forceinline__ void tree_nodes(const TreeParams& p, int* next, bool any) {
  constexpr int V = D / 32, HB = kTreeHeads;
  const int lane = threadIdx.x & 31;
  const int groups = (p.G + HB - 1) / HB, per = p.Hkv * groups, rows_end = next[1];
  for (;;) {
    int turn = 0;
    if (lane == 0) turn = atomicAdd(next, 1);
    const int64_t item = blockIdx.x + int64_t(__shfl_sync(0xffffffffu, turn, 0)) * gridDim.x;
    if (item >= int64_t(rows_end) * per) break;
    const int n = int(item / per), hg = int(item - int64_t(n) * per), h = hg / groups, g0 = (hg - h * groups) * HB;
    const int heads = min(HB, p.G - g0), b = tree_find(p, n);
    const TreeSeq s = tree_seq(p, b);
    const int node = n - s.row0;
    const bool mine = any && !s.bad && node >= 0 && node < s.n;
    const int64_t col0 = int64_t(n) * p.Hq + int64_t(h) * p.G + g0;  // of q, out and the nodes' parts
    float q[HB][V], o[HB][V], m[HB], l[HB];
#pragma unroll
    for (int g = 0; g < HB; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) q[g][i] = o[g][i] = 0.0f;
      if (mine && g < heads)
        load_elements<E, V>(static_cast<const E*>(p.q) + (col0 + g) * D + lane * V, q[g]);
    }
    uint64_t seen = 0;
    int at[2] = {-1, -1};  // rows of nodes lane and lane + 32
    if (mine) {
      seen = p.masks ? uint64_t(__ldcg(reinterpret_cast<const long long*>(p.masks) + n)) : (uint64_t(2) << node) - 1;
      if (s.n < 64) seen &= (uint64_t(1) << s.n) - 1;
      const int64_t place = p.window ? (p.places ? int64_t(__ldcg(p.places + n)) : int64_t(s.held) + node) - p.window : 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = lane + 32 * e;
        bool see = (seen >> j) & 1;
        if (see && p.window) see = (p.places ? __ldcg(p.places + s.row0 + j) : s.held + j) > place;
        if (see) {
          const int t = s.held + j, page = __ldcg(p.tables + int64_t(b) * p.W + t / p.P);
          if (page >= 0 && page < p.n_pages) at[e] = (page * p.Hkv + h) * p.P + (t & (p.P - 1));
          else if (p.flags) atomicOr(p.flags, kErrBadIndex);
        }
        const unsigned v = __ballot_sync(0xffffffffu, see);
        seen = e ? (seen & 0xffffffffull) | (uint64_t(v) << 32) : (seen & ~0xffffffffull) | v;
      }
    }
#pragma unroll 1
    while (seen) {
      StoredPiece<E, BITS, V> kp[8], vp[8];
      bool ok[8];  // alike for all lanes; a page out of range reads as zeros
      int cnt = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        ok[t] = false;
        if (seen) {
          const int j = __ffsll(seen) - 1;
          seen &= seen - 1;
          const int row = __shfl_sync(0xffffffffu, j < 32 ? at[0] : at[1], j & 31);
          ok[t] = row >= 0;
          cnt = t + 1;
          if (ok[t]) {
            kp[t].load(p.k_data, p.k_scales, p.k_biases, row, lane);
            vp[t].load(p.v_data, p.v_scales, p.v_biases, row, lane);
          }
        }
      }
      float sc = -INFINITY;  // of head lane / 8 and token lane % 8
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        float a4[HB] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (ok[t]) {
          float f[V];
          kp[t].get(f);
#pragma unroll
          for (int g = 0; g < HB; ++g)
#pragma unroll
            for (int i = 0; i < V; ++i) a4[g] = fmaf(q[g][i], f[i], a4[g]);
        }
        const bool b4 = lane & 16, b3 = lane & 8;
        float y0 = b4 ? a4[2] : a4[0], y1 = b4 ? a4[3] : a4[1];
        y0 += __shfl_xor_sync(0xffffffffu, b4 ? a4[0] : a4[2], 16);
        y1 += __shfl_xor_sync(0xffffffffu, b4 ? a4[1] : a4[3], 16);
        float y = b3 ? y1 : y0;
        y += __shfl_xor_sync(0xffffffffu, b3 ? y0 : y1, 8);
        y += __shfl_xor_sync(0xffffffffu, y, 4);
        y += __shfl_xor_sync(0xffffffffu, y, 2);
        y += __shfl_xor_sync(0xffffffffu, y, 1);
        if (t < cnt && (lane & 7) == t) sc = y * p.scale_log2;
      }
      float mx = sc;
#pragma unroll
      for (int i = 1; i < 8; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
      float w = 0.0f;
#pragma unroll
      for (int g = 0; g < HB; ++g) {
        const float f = raise_max(m[g], __shfl_sync(0xffffffffu, mx, 8 * g));
        l[g] *= f;
#pragma unroll
        for (int i = 0; i < V; ++i) o[g][i] *= f;
        if (lane >> 3 == g) w = exp2_from(sc, m[g]);
      }
      if ((lane & 7) >= cnt) w = 0.0f;
      float sum = w;
#pragma unroll
      for (int i = 1; i < 8; i <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
#pragma unroll
      for (int g = 0; g < HB; ++g) l[g] += __shfl_sync(0xffffffffu, sum, 8 * g);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        float f[V] = {};
        if (ok[t]) vp[t].get(f);
#pragma unroll
        for (int g = 0; g < HB; ++g) {
          const float pr = __shfl_sync(0xffffffffu, w, 8 * g + t);
          if (ok[t]) {
#pragma unroll
            for (int i = 0; i < V; ++i) o[g][i] = fmaf(pr, f[i], o[g][i]);
          }
        }
      }
    }
#pragma unroll
    for (int g = 0; g < HB; ++g) {
      if (g < heads) {
        float* to = p.node_o + (col0 + g) * D + lane * V;
        if constexpr (V == 4) *reinterpret_cast<float4*>(to) = make_float4(o[g][0], o[g][1], o[g][2], o[g][3]);
        else *reinterpret_cast<float2*>(to) = make_float2(o[g][0], o[g][1]);
        if (lane == 0) p.node_ml[col0 + g] = make_float2(m[g], l[g]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The held tokens
// ---------------------------------------------------------------------------

// The warps of a decode (sd_paged.cuh) with columns for heads, and one for the nodes.
// One pass over the tokens has at most 16 columns, as a decode has heads: bound by
// HBM for few of them, by the conversion of codes and the chain of products beside
// it for 16, by latency for short ranges. Measured with the merge, 32 query and 8 kv
// heads of 128: 16 sequences of 8K tokens, 4 nodes, 8 bits 54 us (2.6 TB/s), 8 of
// them with 2 nodes 32 us; 2K tokens, 7 nodes, fp32, 8 and 2 heads of 64 16 us.
// HELP: the warps come to the nodes' help when they are done. Where a CTA has no second row that only costs (the code
// is larger: 2K tokens and 7 nodes in fp32 take 17.7 us instead of 16.3).
template <typename E, int BITS, int D, int NB, bool HELP>
__global__ void __launch_bounds__(kTreeAttendThreads, 2)
tree_attend_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV) {
  using F = PagedFmt<sizeof(E), BITS, D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* qf = reinterpret_cast<float*>(sm + p.q_off);
  float* buf = reinterpret_cast<float*>(sm + p.buf_off);
  int* units = reinterpret_cast<int*>(sm + p.prefix_off);
  int *pairs = units + p.B + 1, *tmp = pairs + p.B + 1, *low = tmp + 2 * (kTreeAttendThreads / 32), *next = low + kTreeLows;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + p.bar_off);
  uint64_t* empty = full + kPagedMaxStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  static_assert(kTreeCounts == 2 && (NB * (sizeof(E) == 4 && BITS == 0 ? 4 : 8)) <= kTreeLows, "next[0] and next[1]; a token per column");

  if (tid == 0) {
    *next = 0;
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full + i, BITS ? 33 : 1);
      mbar_init(empty + i, kPagedWarps);
    }
    fence_mbar_init();
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  griddep_wait();
  griddep_launch_dependents();
  if (tid == 32) next[1] = min(__ldcg(p.first + p.B), p.N);
  tree_line<kTreeAttendThreads>(p, F::kTile, units, pairs, tmp);  // with barriers

  if (!HELP && warp == kPagedWarps + 1) {
    tree_nodes<E, BITS, D>(p, next, pairs[p.B] > 0);
    return;
  }
  const Pieces pieces(p, units[p.B]);
  if (warp <= kPagedWarps && int(blockIdx.x) < pieces.n) {
    TreeWalk walk(p, units, pairs, pieces.begin(blockIdx.x), pieces.begin(blockIdx.x + 1));
    if (warp == kPagedWarps) {
      paged_produce<E, BITS, D>(p, &tmK, &tmV, sm, full, empty, walk, lane);
    } else {
      using A = typename PickAttend<E, BITS, D, NB, NodeCols>::type;
      const int pb_log = __ffs(min(p.P, F::kTile)) - 1;
      A att;
      TreeSegment s;
      int it = 0, st = 0;
      uint32_t round = 0;
      bool dead = false;
      while (walk.next(s)) {
        const TreeSeq sq = tree_seq(p, s.b);
        const NodeCols cols(p, sq, s.h, s.c);
        const int t0 = sq.begin / F::kTile;
        int edge = 0;  // tokens below it are not seen by every column
        if (p.window) {
          if (tid < kTreeLows) low[tid] = tree_low(p, sq, cols.node(min(tid, cols.n - 1)));
          named_barrier(1, 32 * kPagedWarps);
          edge = __reduce_max_sync(0xffffffffu, low[lane % kTreeLows]);
        }
        att.begin(p, qf, cols, warp, lane);
        for (int i = s.i0; i < s.i1; ++i, ++it) {
          const int tok = (t0 + i) * F::kTile;
          if (!dead) dead = !mbar_wait(full + st, round, p.flags);
          if (!dead) {
            att.tile(p, qf, TileView{sm + st * F::kStageBytes, pb_log, sq.begin - tok, sq.held - tok, tok < edge ? low : nullptr, tok},
                     warp, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + st);
          }
          if (++st == p.stages) {
            st = 0;
            round ^= 1u;
          }
        }
        att.end(cols.n, WarpPart<D>(buf, p.RT, warp), lane);
        named_barrier(1, 32 * kPagedWarps);
        // the four warps' parts, in warp order
        float* part = tree_part(p, s.pair + blockIdx.x);
        for (int k = tid; k < p.RT * (D / 4); k += 32 * kPagedWarps) {
          const int d4 = k / p.RT, g = k - d4 * p.RT;
          if (g >= cols.n) continue;
          float mw[kPagedWarps], M = -INFINITY, L = 0.0f;
#pragma unroll
          for (int w = 0; w < kPagedWarps; ++w) {
            mw[w] = WarpPart<D>(buf, p.RT, w).ml[2 * g];
            M = fmaxf(M, mw[w]);
          }
          float4 O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int w = 0; w < kPagedWarps; ++w) {
            const WarpPart<D> wp(buf, p.RT, w);
            const float f = exp2_from(mw[w], M);
            const float4 x = *reinterpret_cast<const float4*>(wp.o + g * (D + 4) + 4 * d4);
            L = fmaf(f, wp.ml[2 * g + 1], L);
            O.x = fmaf(f, x.x, O.x);
            O.y = fmaf(f, x.y, O.y);
            O.z = fmaf(f, x.z, O.z);
            O.w = fmaf(f, x.w, O.w);
          }
          reinterpret_cast<float4*>(part)[k] = O;
          if (d4 == 0) *reinterpret_cast<float2*>(part + p.RT * D + 2 * g) = make_float2(M, L);
        }
        named_barrier(1, 32 * kPagedWarps);
      }
      if (dead) drain(full, it, p.stages);
    }
  }
  if constexpr (HELP) tree_nodes<E, BITS, D>(p, next, pairs[p.B] > 0);
}

// Of one kv head, kTreeMergeCols neighbouring columns (row, query head) per
// block: a thread has one column and four dimensions, and eight segments' loads
// under way. Bound by latency: the line, the segments' places, their loads. Alone
// and with cold caches it takes 10 us for 1024 columns of 128 and 18 us for 8192.
template <typename E, int D>
__global__ void __launch_bounds__(kTreeMergeCols * D / 4) tree_merge_kernel(const __grid_constant__ TreeParams p) {
  constexpr int NC = kTreeMergeCols;
  const int columns = p.N * p.G, blocks = (columns + NC - 1) / NC, h = blockIdx.x / blocks;
  const int col = threadIdx.x % NC, d4 = threadIdx.x / NC, x = (blockIdx.x - h * blocks) * NC + col;
  const int n = p.by_g(min(x, columns - 1)), g = x - n * p.G;
  const bool live = x < columns && n < __ldcg(p.first + p.B);  // rows behind the last sequence stay as they are
  int b = 0;
  TreeSeq s{};
  if (live) {
    b = tree_find(p, n);
    s = tree_seq(p, b);
  }
  griddep_wait();
  if (!live) return;
  const int64_t row = int64_t(n) * p.Hq + int64_t(h) * p.G + g;
  float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float M = -INFINITY, L = 0.0f;
  if (p.node_ml) {
    const float2 ml = __ldcg(p.node_ml + row);
    M = ml.x, L = ml.y;
    O = __ldcg(reinterpret_cast<const float4*>(p.node_o + row * D) + d4);
  }
  const int i = n - s.row0;
  int up = 0, u1 = 0, all = 0, pp = 0, np = 0;
  if (i >= 0 && i < s.n && s.end > s.begin) {
    up = __ldcg(p.line + b), u1 = __ldcg(p.line + b + 1), all = __ldcg(p.line + p.B);
    pp = __ldcg(p.line + p.B + 1 + b), np = __ldcg(p.line + p.B + 2 + b) - pp;
  }
  if (np > 0) {
    const int nu = (u1 - up) / np, y = i * p.G + g, c = y / p.RT, k = h * (np / p.Hkv) + c, at = y - c * p.RT;
    const Pieces pieces(p, all);
    const int a = up + k * nu, cta = pieces.of(a + p.seg_units), ns = pieces.of(a + nu - 1) - cta + 1;
    const float* part = tree_part(p, pp + k + cta);
#pragma unroll 1
    for (int j0 = 0; j0 < ns; j0 += 8) {
      float2 ml[8];
      float4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ml[j] = make_float2(-INFINITY, 0.0f);
        v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (j0 + j < ns) {
          const float* from = part + int64_t(j0 + j) * p.part_floats;
          ml[j] = __ldcg(reinterpret_cast<const float2*>(from + p.RT * D) + at);
          v[j] = __ldcg(reinterpret_cast<const float4*>(from) + d4 * p.RT + at);
        }
      }
      float top = ml[0].x;
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, ml[j].x);
      const float f = raise_max(M, top);
      L *= f;
      O.x *= f, O.y *= f, O.z *= f, O.w *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = exp2_from(ml[j].x, M);
        L = fmaf(w, ml[j].y, L);
        O.x = fmaf(w, v[j].x, O.x), O.y = fmaf(w, v[j].y, O.y);
        O.z = fmaf(w, v[j].z, O.z), O.w = fmaf(w, v[j].w, O.w);
      }
    }
  }
  if (p.sinks) L += exp2f(fmaf(__ldcg(p.sinks + h * p.G + g), 1.4426950408889634f, -(M == -INFINITY ? 0.0f : M)));
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  E* out = static_cast<E*>(p.out) + row * D + 4 * d4;
  if constexpr (sizeof(E) == 4) *reinterpret_cast<float4*>(out) = make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
  else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<E>(O.x * inv, O.y * inv), pack2<E>(O.z * inv, O.w * inv));
}

}  // namespace sd
