// sd_draft.cu -- the plan of a step of new tokens, and the rows that stay of
// them.
#include "sd_device.cuh"
#include "sd_draft.h"

namespace sd {

namespace {

// Exclusive sum of v over the block's threads in order; *total: of all.
__device__ __forceinline__ int64_t block_before(int64_t v, int64_t* sums, int64_t* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  int64_t incl = v;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, x);
    if (lane >= x) incl += y;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < nw; ++w) {
    before += w < warp ? sums[w] : 0;
    all += sums[w];
  }
  __syncthreads();
  *total = all;
  return before + incl - v;
}

template <typename T>
__device__ __forceinline__ void store4(T* at, int64_t row, int n, const T (&v)[kPlanRows], bool wide) {
  if (wide && n == kPlanRows) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<int4*>(at + row) = make_int4(v[0], v[1], v[2], v[3]);
    } else {
      *reinterpret_cast<longlong2*>(at + row) = make_longlong2(v[0], v[1]);
      *reinterpret_cast<longlong2*>(at + row + 2) = make_longlong2(v[2], v[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPlanRows; ++i)
      if (i < n) at[row + i] = v[i];
  }
}

}  // namespace

// Sequence b has len[b] tokens and gets n[b] more. With c[b] pages held,
//   need[b] = max(0, ceil((len + n) / P) - c), from free[taken + sum_{a < b} need[a]] on,
// rows first[b] = sum_{a < b} n[a] on are its new tokens: row first[b] + i lies at
// position len[b] + i, slot table[position / P] * P + position % P. Of a tree,
// node i's mask has its own bit and those of its parent's mask, its place is
// one past its parent's (the sequence's length for a root). What does not fit
// (the table, the free pages, the tree, the rows) is cut, with an error bit,
// so that what is planned can always be done; a sequence with more tokens than its
// table holds gets nothing, so no page is written behind a table's row.
//
// Bound by latency up to some ten thousand rows (a launch, the lengths, the
// table), then by its stores: 16 bytes a row, 28 with a tree. Every CTA works out all sequences'
// sums for itself (at most 4096) and then takes blocks of rows; a thread
// finds its first row's sequence by bisection and goes on from there. Of trees a
// warp takes a whole one: lane l has nodes l and l + 32, and six exchanges, each
// of which doubles how far up a node has looked, make every mask (a walk up by
// one load per ancestor took 50 us for 64 trees of 32). The pages taken are
// written by the same launch where its CTAs can wait until all have read what
// is held (one cluster of at most 8), and by a second one otherwise, page by page:
// neighbouring threads have neighbouring entries of the list.
// Measured, launches in a graph: one token 2.8 us, 64 trees of 32 nodes 4.4 us,
// 512 prompts of 2000 tokens 13 us (16.6 MB, 1.3 TB/s; it waits for bisections and
// tables as much as for stores) and 23 us where they take their 64K pages.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int sm[];
  __shared__ int64_t sums[kPlanThreads / 32];
  int *first = sm, *len = first + p.B + 1, *have = len + p.B, *base = have + p.B;
  const int tid = threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();

  const int per = (p.B + kPlanThreads - 1) / kPlanThreads, b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  const int taken = p.held ? max(0, min(__ldcg(p.taken), p.n_free)) : 0;
  bool bad = p.held && taken != __ldcg(p.taken);
  // first[b + 1]: the new tokens of b, as far as the table and the tree hold them
  int64_t need = 0;
  for (int b = b0; b < b1; ++b) {
    const int raw = __ldcg(p.lengths + b), add = __ldcg(p.added + b);
    const int l = max(raw, 0), c = p.held ? __ldcg(p.held + b) : p.W, h = max(0, min(c, p.W));
    const bool past = l > int64_t(p.W) * p.P;  // more tokens than the table holds: neither tokens nor pages
    int n = int(max(int64_t(0), min(int64_t(max(add, 0)), min(int64_t(p.W) * p.P - l, int64_t(p.N)))));
    if (p.parents) n = min(n, p.T);
    bad = bad || raw < 0 || n != add || h != c || past;
    len[b] = l;
    have[b] = h;
    first[b + 1] = n;
    base[b] = max(0, int((int64_t(l) + n + p.P - 1) >> p.page_shift) - h);
    if (!p.held || past) base[b] = 0;
    need += base[b];
  }
  int64_t all, run = block_before(need, sums, &all);
  need = 0;  // from here on: rows
  for (int b = b0; b < b1; ++b) {
    const int want = base[b], got = int(max(int64_t(0), min(int64_t(want), p.n_free - taken - run)));
    base[b] = int(min(run, int64_t(p.n_free - taken))) + taken;
    run += want;
    if (got < want) {
      bad = true;
      first[b + 1] = int(max(int64_t(0), min(int64_t(first[b + 1]), (int64_t(have[b]) + got) * p.P - len[b])));
    }
    need += first[b + 1];
  }
  const int pages_end = int(min(all, int64_t(p.n_free - taken))) + taken;
  run = block_before(need, sums, &all);
  for (int b = b0; b < b1; ++b) {
    const int n = first[b + 1];
    bad = bad || run + n > p.N;
    run += n;
    first[b + 1] = int(min(run, int64_t(p.N)));
  }
  if (tid == 0) first[0] = 0;
  __syncthreads();
  const int total = first[p.B];
  if (bad && p.flags && blockIdx.x == 0) atomicOr(p.flags, kErrBadIndex);

  if (p.rows) {
    for (int b = blockIdx.x * kPlanThreads + tid; b <= p.B; b += gridDim.x * kPlanThreads) {
      p.first[b] = first[b];
      if (b < p.B) p.ends[b] = len[b] + first[b + 1] - first[b];
    }
    const bool wide = ((reinterpret_cast<uintptr_t>(p.seq) | reinterpret_cast<uintptr_t>(p.positions) |
                        reinterpret_cast<uintptr_t>(p.places) | reinterpret_cast<uintptr_t>(p.slots) |
                        reinterpret_cast<uintptr_t>(p.masks)) & 15) == 0;
    // page and slot of position `at` of sequence b
    auto slot_of = [&](int b, int at) {
      const int col = at >> p.page_shift;
      const int page = col < have[b] ? __ldcg(p.tables + int64_t(b) * p.W + col) : __ldcg(p.free_pages + base[b] + col - have[b]);
      return page < 0 ? int64_t(-1) : int64_t(page) * p.P + (at & (p.P - 1));
    };
    if (p.parents) {
      const int lane = tid & 31, warps = gridDim.x * (kPlanThreads / 32);
      bool odd = false;  // a parent that does not come before its node
      for (int b = blockIdx.x * (kPlanThreads / 32) + (tid >> 5); b < p.B; b += warps) {
        const int n = first[b + 1] - first[b];
        const int* up = p.parents + b * p.parents_stride;
        uint32_t lo[2], hi[2];  // the masks' words
        int next[2];            // the ancestor to look at from; -1: none, -2: there is no such node
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int node = lane + 32 * e;
          next[e] = node < n ? __ldcg(up + node) : -2;
          odd |= node < n && next[e] >= node;
          if (next[e] < -1 || next[e] >= node) next[e] = -2;
          lo[e] = e ? 0u : 1u << lane, hi[e] = e ? 1u << lane : 0u;
        }
        while (__any_sync(0xffffffffu, next[0] >= 0 || next[1] >= 0)) {  // six times at most
          uint32_t l2[2], h2[2];
          int n2[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int from = max(next[e], 0), at = from & 31;
            const bool far = from >= 32;
            const uint32_t a = __shfl_sync(0xffffffffu, lo[0], at), c = __shfl_sync(0xffffffffu, lo[1], at);
            const uint32_t d = __shfl_sync(0xffffffffu, hi[0], at), f = __shfl_sync(0xffffffffu, hi[1], at);
            const int g = __shfl_sync(0xffffffffu, next[0], at), k = __shfl_sync(0xffffffffu, next[1], at);
            l2[e] = far ? c : a, h2[e] = far ? f : d, n2[e] = far ? k : g;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (next[e] >= 0) lo[e] |= l2[e], hi[e] |= h2[e], next[e] = n2[e];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int node = lane + 32 * e;
          if (node >= n) continue;
          const int64_t r = first[b] + node;
          const bool there = next[e] == -1;
          p.seq[r] = b;
          p.positions[r] = there ? len[b] + node : -1;
          if (p.slots) p.slots[r] = there ? slot_of(b, len[b] + node) : -1;
          if (p.places) p.places[r] = there ? len[b] + __popc(lo[e]) + __popc(hi[e]) - 1 : -1;
          if (p.masks) p.masks[r] = there ? int64_t(uint64_t(hi[e]) << 32 | lo[e]) : 0;
        }
      }
      for (int64_t r = int64_t(total) + blockIdx.x * kPlanThreads + tid; r < p.N; r += int64_t(gridDim.x) * kPlanThreads) {
        p.seq[r] = p.positions[r] = -1;
        if (p.slots) p.slots[r] = -1;
        if (p.places) p.places[r] = -1;
        if (p.masks) p.masks[r] = 0;
      }
      if (odd && p.flags) atomicOr(p.flags, kErrBadIndex);
    }
    const int64_t step = int64_t(gridDim.x) * kPlanThreads * kPlanRows;
    for (int64_t r0 = (int64_t(blockIdx.x) * kPlanThreads + tid) * kPlanRows; r0 < p.N && !p.parents; r0 += step) {
      const int cnt = int(min(int64_t(kPlanRows), p.N - r0));
      int seq[kPlanRows], pos[kPlanRows], place[kPlanRows];
      int64_t slot[kPlanRows], mask[kPlanRows];
      int b = 0;
      if (r0 < total) {  // the last b with first[b] <= r0: it has rows
        int hi = p.B;
        while (hi - b > 1) {
          const int mid = (b + hi) >> 1;
          if (first[mid] <= r0) b = mid; else hi = mid;
        }
      }
#pragma unroll
      for (int i = 0; i < kPlanRows; ++i) {
        const int r = int(r0) + i;
        seq[i] = pos[i] = place[i] = -1;
        slot[i] = -1;
        mask[i] = 0;
        if (i >= cnt || r >= total) continue;
        while (r >= first[b + 1]) ++b;  // ends: r < total
        const int node = r - first[b], at = len[b] + node;
        seq[i] = b;
        pos[i] = place[i] = at;
        mask[i] = int64_t((uint64_t(2) << min(node, kMaxNodes - 1)) - 1);
        slot[i] = slot_of(b, at);
      }
      store4(p.seq, r0, cnt, seq, wide);
      store4(p.positions, r0, cnt, pos, wide);
      if (p.slots) store4(p.slots, r0, cnt, slot, wide);
      if (p.places) store4(p.places, r0, cnt, place, wide);
      if (p.masks) store4(p.masks, r0, cnt, mask, wide);
    }
  }
  if (!p.commit) return;
  if (gridDim.x > 1) cluster_sync();  // every CTA has read what is held
  for (int b = blockIdx.x * kPlanThreads + tid; b < p.B; b += gridDim.x * kPlanThreads) {
    const int got = (b + 1 < p.B ? base[b + 1] : pages_end) - base[b];
    if (got > 0) p.held[b] = have[b] + got;
  }
  // kPlanRows neighbouring pages of the list per thread
  for (int64_t j0 = taken + (blockIdx.x * kPlanThreads + tid) * kPlanRows; j0 < pages_end;
       j0 += gridDim.x * kPlanThreads * kPlanRows) {
    int page[kPlanRows], b = 0, hi = p.B;
#pragma unroll
    for (int i = 0; i < kPlanRows; ++i)
      if (j0 + i < pages_end) page[i] = __ldcg(p.free_pages + j0 + i);
    while (hi - b > 1) {  // the last b with base[b] <= j0: it takes pages
      const int mid = (b + hi) >> 1;
      if (base[mid] <= j0) b = mid; else hi = mid;
    }
#pragma unroll
    for (int i = 0; i < kPlanRows; ++i) {
      if (j0 + i >= pages_end) break;
      while (b + 1 < p.B && base[b + 1] <= j0 + i) ++b;
      p.tables[int64_t(b) * p.W + have[b] + j0 + i - base[b]] = page[i];
    }
  }
  if (blockIdx.x == 0 && tid == 0) *p.taken = pages_end;
}

const void* plan_kernel_ptr() { return reinterpret_cast<const void*>(&plan_kernel); }

namespace {

// Rows src[i] -> dst[i] (row numbers of head 0, -1: stays), i < n, of one column of an array: W bytes at `at`.
template <typename W>
__device__ __forceinline__ void keep_rows(uint8_t* at, int row, const int* src, const int* dst, int n) {
  for (int i0 = 0; i0 < n; i0 += kKeepBatch) {
    W x[kKeepBatch];
#pragma unroll
    for (int i = 0; i < kKeepBatch; ++i)
      if (i0 + i < n && src[i0 + i] >= 0) x[i] = *reinterpret_cast<const W*>(at + int64_t(src[i0 + i]) * row);
#pragma unroll
    for (int i = 0; i < kKeepBatch; ++i)
      if (i0 + i < n && src[i0 + i] >= 0) *reinterpret_cast<W*>(at + int64_t(dst[i0 + i]) * row) = x[i];
  }
}

}  // namespace

// Row h + i of a sequence becomes its row h + path[i], i < kept, in every layer,
// K and V (h: its tokens before the step), and its length h + kept. path rises,
// so path[i] >= i: a row is overwritten only when it has been read, if rows are
// taken in order -- a thread does so with its own 16 bytes of a (head, row),
// eight rows under way at a time, and no thread waits for another. One block
// per (layer, sequence). Bound by HBM for many users, by latency (path, table,
// rows: three loads one after the other) for few. Measured in a graph, 36 layers of
// 8 kv heads of 128: one user's 16 nodes in bf16 3.0 us (1.2 MB), 64 users' of 32 in
// 8 bits 13 us (16.6 MB, 1.3 TB/s: 2304 short blocks, most of whose time is that chain).
__global__ void __launch_bounds__(kKeepThreads) keep_kernel(const __grid_constant__ KeepParams p) {
  __shared__ int src[kMaxNodes], dst[kMaxNodes], count;
  const int tid = threadIdx.x, b = blockIdx.x % p.B, layer = blockIdx.x / p.B;
  griddep_wait();
  griddep_launch_dependents();
  if (tid < 32) {
    const int f0 = __ldcg(p.first + b), f1 = __ldcg(p.first + b + 1), end = __ldcg(p.ends + b), k0 = __ldcg(p.kept + b);
    int64_t nodes = int64_t(f1) - f0, held = int64_t(end) - nodes;
    bool bad = false;
    if (nodes < 0 || held < 0 || end > int64_t(p.W) * p.P) {
      bad = true;
      nodes = 0;
      held = max(int64_t(0), min(int64_t(end), int64_t(p.W) * p.P));
    }
    int k = int(max(int64_t(0), min(int64_t(k0), min(int64_t(p.T), nodes))));
    bad = bad || k != k0;
    int stop = k;  // the first entry that cannot be done
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = half * 32 + tid;
      bool wrong = false;
      if (i < k) {
        const int* path = p.path + int64_t(b) * p.T;
        const int j = __ldcg(path + i), before = i ? __ldcg(path + i - 1) : -1;
        wrong = j <= before || j >= nodes;
        int from = -1, to = -1;
        if (!wrong && j != i) {
          const int a = int(held) + j, c = int(held) + i;
          const int pa = __ldcg(p.tables + int64_t(b) * p.W + (a >> p.page_shift));
          const int pc = __ldcg(p.tables + int64_t(b) * p.W + (c >> p.page_shift));
          wrong = pa < 0 || pa >= p.n_pages || pc < 0 || pc >= p.n_pages;
          if (!wrong) {
            from = pa * p.Hkv * p.P + (a & (p.P - 1));
            to = pc * p.Hkv * p.P + (c & (p.P - 1));
          }
        }
        src[i] = from;
        dst[i] = to;
      }
      const unsigned w = __ballot_sync(0xffffffffu, wrong);
      if (w) stop = min(stop, half * 32 + __ffs(w) - 1);
    }
    if (stop < k) bad = true;
    if (tid == 0) {
      count = stop;
      if (layer == 0) {
        p.lengths[b] = int(held) + stop;
        if (bad && p.flags) atomicOr(p.flags, kErrBadIndex);
      }
    }
  }
  __syncthreads();
  const int n = count;
  for (int c = tid; c < p.all_columns && n > 0; c += kKeepThreads) {
    int a = 0, x = c;
#pragma unroll
    for (int i = 0; i < 5; ++i)
      if (a == i && x >= p.columns[i]) x -= p.columns[i], ++a;
    const int row = p.row[a], width = min(row, 16), per = row / width;
    const int h = x / per;
    uint8_t* at = p.array[a] + p.layer[a] * layer + int64_t(h) * p.P * row + (x - h * per) * width;
    switch (width) {
      case 16: keep_rows<uint4>(at, row, src, dst, n); break;
      case 8: keep_rows<uint2>(at, row, src, dst, n); break;
      case 4: keep_rows<uint32_t>(at, row, src, dst, n); break;
      default: keep_rows<uint16_t>(at, row, src, dst, n);
    }
  }
}

const void* keep_kernel_ptr() { return reinterpret_cast<const void*>(&keep_kernel); }

}  // namespace sd
