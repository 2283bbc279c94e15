// sd_tree_tile.cu -- attention of many (node, query head) columns per sequence
// to the held tokens of 16-bit pools, on the fifth-generation tensor cores.
// See sd_tree.cuh for what it is a part of.
//
// A pair's columns are the rows of 128-row accumulators: S = Q K^T (128 rows x
// 128 tokens), P = 2^(S - m), O += P V. S and O live in tensor memory, P takes
// S's place there as the next product's left operand, Q, K and V are 128B-
// swizzled tiles in shared memory (TMA, one box per page and 64 dimensions).
// One warp loads, one thread issues the products, and two groups of four warps
// hold a row per thread and make P, each with its own S and O, so that the
// products of one group run while the other makes its P:
//   SHARED: the pair has up to 256 columns, 128 per group, and both groups use
//     every tile;
//   else: it has up to 128, both groups have the same ones, and tiles go to the
//     groups in turn, whose parts are joined at a segment's end.
// P is one value of the element type: 128 x 128 products cost as much as their
// exponentials, and a second half would cost as much again (SHARED). The sum
// that O is divided by is made of the rounded values, so their errors cancel
// where few tokens have the weight.
//
// The running maximum lags by up to kSlack, as in a decode; when it moves, its
// group rescales O in tensor memory. Rows of V outside the range may hold
// anything and are zeroed in shared memory (0 * NaN is NaN); scores there are
// replaced.
#include "sd_tree.cuh"

namespace sd {

namespace {

constexpr int kTileT = kTreeTileTokens;
constexpr int kTmemCols = 512;
constexpr int kSCol = 0, kOCol = 256;  // tensor memory columns of the first group's S and O; the second's 128 on

// --- tensor core pieces -----------------------------------------------------

// Shared-memory operand descriptor, 128-byte swizzle; lead / stride: byte offsets (see the operand's layout).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return uint64_t((addr >> 4) & 0x3fff) | (uint64_t((lead >> 4) & 0x3fff) << 16) | (uint64_t((stride >> 4) & 0x3fff) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor: fp32 accumulator, 16-bit operands, M = 128; b_mn: B's rows are contiguous along N.
template <typename E>
__host__ __device__ constexpr uint32_t product_desc(int n, bool b_mn) {
  constexpr uint32_t fmt = __is_same(E, __half) ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(int(add))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(int(add))
      : "memory");
}
// The barrier gets one arrival when the products issued so far by this thread are done.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define SD_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define SD_W8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
// 32 columns of this warp's 32 lanes; v: the thread's row.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : SD_R8(v, 0), SD_R8(v, 8), SD_R8(v, 16), SD_R8(v, 24)
      : "r"(addr));
}
// The loads before are done; the operands keep what uses v behind it.
#define SD_U8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
__device__ __forceinline__ void tmem_wait(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : SD_U8(v, 0), SD_U8(v, 8), SD_U8(v, 16), SD_U8(v, 24)::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
               SD_W8(v, 0), SD_W8(v, 8)
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      SD_W8(v, 0), SD_W8(v, 8), SD_W8(v, 16), SD_W8(v, 24)
      : "memory");
}

// --- waits: bounded; the answer is the warp's, as the tensor memory accesses are ---
struct Waiter {
  int* flags;
  bool dead;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) {
    if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity, flags));
    return !dead;
  }
};

struct TileBars {
  uint64_t full[kTreeTileStages], empty[kTreeTileStages];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], done;
  uint32_t tmem;
};
static_assert(sizeof(TileBars) <= kTreeTileBarBytes, "room in the layout");

}  // namespace

template <typename E, int D, bool SHARED>
__global__ void __launch_bounds__(kTreeTileThreads, 1)
tree_tile_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV) {
  constexpr int NH = D / 64, kHalf = 128 * 128, kStage = NH * kHalf;  // bytes: 128 rows x 64 elements; a tile of K or V
  constexpr float kUp = __is_same(E, __half) ? 7.0f : 0.0f;  // as in a decode: fp16 weights up to 2^(kUp + kSlack)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *qs = sm, *ring = sm + 2 * kStage;
  TileBars* bars = reinterpret_cast<TileBars*>(sm + p.bar_off);
  int* units = reinterpret_cast<int*>(sm + p.prefix_off);
  int *pairs = units + p.B + 1, *tmp = pairs + p.B + 1;
  __shared__ float2 other[SHARED ? 1 : 128];  // (m, l) of the second group
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(bars->full + i, 1);
      mbar_init(bars->empty + i, 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(bars->q_full + w, 128);
      mbar_init(bars->s_full + w, 1);
      mbar_init(bars->p_full + w, 128);
      mbar_init(bars->o_full + w, 1);
    }
    mbar_init(&bars->done, 1);
    fence_mbar_init();
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  griddep_wait();
  griddep_launch_dependents();
  tc_fence_before();
  tree_line<kTreeTileThreads>(p, kTileT, units, pairs, tmp);  // with barriers
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  const Pieces pieces(p, units[p.B]);
  const bool work = int(blockIdx.x) < pieces.n;
  TreeWalk walk(units, pairs, p.B, p.Hkv, work ? pieces.begin(blockIdx.x) : 0, work ? pieces.begin(blockIdx.x + 1) : 0);
  TreeSegment s;
  int it0 = 0;  // tiles of the segments before
  Waiter wait{p.flags, false};

  if (warp == 8) {  // ---- loads ----
    const uint64_t pol = stream_policy(false);
    const int pb = min(p.P, kTileT), nb = kTileT / pb;  // rows per box, boxes per tile
    const int p_log = __ffs(p.P) - 1;
    const int oob_row = int(p.n_pages * p.Hkv * p.P);  // past the tensor: TMA fills zeros
    int use = 0, st = 0;  // stages used so far, the next one
    uint32_t round = 0;
    while (walk.next(s)) {
      const TreeSeq sq = tree_seq(p, s.b);
      const int* row = p.tables + int64_t(s.b) * p.W;
      const int t0 = sq.begin / kTileT, last_slot = (sq.held - 1) >> p_log, first_slot = sq.begin >> p_log;
      auto load = [&](int slot) { return slot >= first_slot && slot <= last_slot ? row[slot] : -1; };
      int base = ((t0 + s.i0) * kTileT) >> p_log;
      int cur = load(base + lane), nxt = load(base + 32 + lane);
      for (int i = s.i0; i < s.i1 && !wait.dead; ++i) {
        const int tok = (t0 + i) * kTileT;
        if ((tok >> p_log) - base >= 32) {
          base += 32;
          cur = nxt;
          nxt = load(base + 32 + lane);
        }
        const int tj = tok + (lane < nb ? lane : 0) * pb, off = (tj >> p_log) - base;
        const int a = __shfl_sync(0xffffffffu, cur, off & 31), c = __shfl_sync(0xffffffffu, nxt, off & 31);
        const int page = off < 32 ? a : c;
        const bool need = lane < nb && tj < sq.held && tj + pb > sq.begin;
        int y = oob_row;
        if (need) {
          if (page >= 0 && page < p.n_pages) y = int((int64_t(page) * p.Hkv + s.h) * p.P + (tj & (p.P - 1)));
          else if (p.flags) atomicOr(p.flags, kErrBadIndex);
        }
        const int n_box = __popc(__ballot_sync(0xffffffffu, need));
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (use >= p.stages && !wait(bars->empty + st, round ^ 1u)) break;
          uint64_t* full = bars->full + st;
          if (lane == 0) mbar_arrive_expect_tx(full, uint32_t(n_box * NH * pb * 128));
          __syncwarp();
          if (need) {
            uint8_t* dst = ring + st * kStage + lane * pb * 128;
#pragma unroll
            for (int h = 0; h < NH; ++h) tma_load_3d(dst + h * kHalf, kv ? &tmV : &tmK, 0, y, h, full, pol);
          }
          ++use;
          if (++st == p.stages) {
            st = 0;
            round ^= 1u;
          }
        }
      }
    }
    if (wait.dead)  // what is under way lands in this CTA's shared memory
      for (int u = max(0, use - p.stages); u < use; ++u) mbar_wait(bars->full + u % p.stages, uint32_t(u / p.stages) & 1u, nullptr);
  } else if (warp == 9) {  // ---- products ----
    uint32_t seg[2] = {0, 0}, k[2] = {0, 0};  // segments and steps of each group: the parities of its barriers
    const uint32_t ring_a = smem_u32(ring);
    const uint32_t first_lane = lane == 0;
    while (walk.next(s)) {
      const int nt = s.i1 - s.i0, n = SHARED ? 2 * nt : nt;
      auto stage_of = [&](int step, int kv) { return 2 * (it0 + (SHARED ? step >> 1 : step)) + kv; };
      auto landed = [&](int u) { return wait(bars->full + u % p.stages, uint32_t(u / p.stages) & 1u); };
      auto scores = [&](int step) {  // S of a step
        const int w = step & 1, u = stage_of(step, 0);
        if (!landed(u)) return;
        tc_fence_after();
        if (first_lane) {
          const uint32_t q = smem_u32(qs) + w * kStage, kk = ring_a + (u % p.stages) * kStage;
#pragma unroll
          for (int c = 0; c < D / 16; ++c)
            mma_ss(tmem + kSCol + w * 128, operand_desc(q + (c / 4) * kHalf + (c % 4) * 32, 16, 1024),
                   operand_desc(kk + (c / 4) * kHalf + (c % 4) * 32, 16, 1024), product_desc<E>(kTileT, false), c > 0);
          mma_commit(bars->s_full + w);
          if (!SHARED || w == 1) mma_commit(bars->empty + u % p.stages);
        }
        __syncwarp();
      };
      // A group with steps loads its rows of Q first, and has read what it needs of its last S and O then. One without
      // (a segment of one tile) does not take part: it could run ahead of this wait by more than a phase.
      for (int w = 0; w < min(n, 2); ++w, ++seg[w - 1])
        if (wait(bars->q_full + w, seg[w] & 1u)) scores(w);
      for (int step = 0; step < n && !wait.dead; ++step) {
        const int w = step & 1, u = stage_of(step, 1);
        if (!wait(bars->p_full + w, k[w] & 1u) || !landed(u)) break;
        tc_fence_after();
        if (first_lane) {
          const uint32_t v = ring_a + (u % p.stages) * kStage;
#pragma unroll
          for (int c = 0; c < kTileT / 16; ++c)
            mma_ts(tmem + kOCol + w * 128, tmem + kSCol + w * 128 + c * 8, operand_desc(v + c * 2048, kHalf, 1024),
                   product_desc<E>(D, true), step > 1 || c > 0);
          mma_commit(bars->o_full + w);
          if (!SHARED || w == 1) mma_commit(bars->empty + u % p.stages);
        }
        __syncwarp();
        if (step + 2 < n) {
          if (!wait(bars->o_full + w, k[w] & 1u)) break;  // P lies where the next S goes
          scores(step + 2);
        }
        ++k[w];
      }
      it0 += nt;
    }
    if (first_lane) mma_commit(&bars->done);  // no product may read shared memory that is no longer this CTA's
    __syncwarp();
    mbar_wait(&bars->done, 0, p.flags);
  } else {  // ---- weights: a row per thread ----
    const int w = warp >> 2, r = tid & 127;  // group, row in it
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // the 32 lanes of tensor memory that this warp reaches
    const uint32_t ts = tmem + lanes + kSCol + w * 128, to = tmem + lanes + kOCol + w * 128;
    const bool neg = p.scale_log2 < 0.0f;
    const float sc = fmaxf(fabsf(p.scale_log2), 1.1754944e-38f);  // -inf times it stays -inf
    uint32_t k = 0;  // steps of this group
    while (walk.next(s)) {
      const TreeSeq sq = tree_seq(p, s.b);
      const NodeCols cols(p, sq, s.h, s.c);
      const int x = SHARED ? w * 128 + r : r;  // column of the pair
      const int t0 = sq.begin / kTileT;
      const int low = p.window && x < cols.n ? tree_low(p, sq, cols.node(x)) : 0;
      const int edge = __reduce_max_sync(0xffffffffu, low);
      if (SHARED || s.i0 + w < s.i1) {  // Q: 16 bytes at a time, a row's chunks side by side
        constexpr int CPR = D / 8;
        const uint32_t q = smem_u32(qs) + w * kStage;
#pragma unroll 4
        for (int c = r; c < 128 * CPR; c += 128) {
          const int row = c / CPR, ch = c % CPR, xx = (SHARED ? w * 128 : 0) + row;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (xx < cols.n) v = __ldcg(reinterpret_cast<const uint4*>(static_cast<const E*>(p.q) + cols.row(xx) * D) + ch);
          const uint32_t at = q + (ch / 8) * kHalf + row * 128 + (((ch % 8) ^ (row & 7)) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }
        fence_proxy_async_shared();
        tc_fence_before();
        mbar_arrive(bars->q_full + w);
      }
      float m = -INFINITY, l = 0.0f;
      int steps = 0;
      for (int i = s.i0 + (SHARED ? 0 : w); i < s.i1; i += SHARED ? 1 : 2, ++steps, ++k) {
        const int tok = (t0 + i) * kTileT, lo = sq.begin - tok, hi = sq.held - tok;
        if (!wait(bars->s_full + w, k & 1u)) continue;
        tc_fence_after();
        // The row's scores, 32 at a time, twice: for the maximum and for the weights. All 128 in registers would spill.
        const bool some = lo > 0 || hi < kTileT || tok < edge;  // some may not be seen
        const int from = max(lo, low - tok);
        auto as_seen = [&](uint32_t (&v)[32], int c) {
          if (neg) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] ^= 0x80000000u;
          }
          if (some) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 32 * c + j < from || 32 * c + j >= hi ? 0xff800000u : v[j];
          }
        };
        uint32_t va[32], vb[32];
        float mx[2] = {-INFINITY, -INFINITY};
        auto most = [&](uint32_t (&v)[32], int c) {
          as_seen(v, c);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            mx[0] = fmaxf(mx[0], __uint_as_float(v[j]));
            mx[1] = fmaxf(mx[1], __uint_as_float(v[j + 1]));
          }
        };
        tmem_ld32(ts, va);
        tmem_wait(va);
        tmem_ld32(ts + 32, vb);
        most(va, 0);
        tmem_wait(vb);
        tmem_ld32(ts + 64, va);
        most(vb, 1);
        tmem_wait(va);
        tmem_ld32(ts + 96, vb);
        most(va, 2);
        tmem_wait(vb);
        tmem_ld32(ts, va);
        most(vb, 3);
        const float top = fmaxf(mx[0], mx[1]) * sc;
        if (steps == 0) {
          m = top - kUp;
        } else if (__any_sync(0xffffffffu, top > m + (kSlack + kUp))) {
          const float fac = raise_max(m, top - kUp);
          l *= fac;
          if (wait(bars->o_full + w, (k - 1) & 1u)) {
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              tmem_ld32(to + 32 * c, vb);
              tmem_wait(vb);
#pragma unroll
              for (int j = 0; j < 32; ++j) vb[j] = __float_as_uint(__uint_as_float(vb[j]) * fac);
              tmem_st32(to + 32 * c, vb);
            }
          }
        }
        const float mm = m == -INFINITY ? 0.0f : m;
        float sum[2] = {0.0f, 0.0f};
        auto weigh = [&](uint32_t (&v)[32], int c) {  // P takes the place of scores that have been read
          as_seen(v, c);
          uint32_t two[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            two[j] = pack2<E>(ex2(fmaf(__uint_as_float(v[2 * j]), sc, -mm)), ex2(fmaf(__uint_as_float(v[2 * j + 1]), sc, -mm)));
            float g[2];
            unpack_word<E>(two[j], g);
            sum[0] += g[0];
            sum[1] += g[1];
          }
          tmem_st16(ts + 16 * c, two);
        };
        tmem_wait(va);
        tmem_ld32(ts + 32, vb);
        weigh(va, 0);
        tmem_wait(vb);
        tmem_ld32(ts + 64, va);
        weigh(vb, 1);
        tmem_wait(va);
        tmem_ld32(ts + 96, vb);
        weigh(va, 2);
        tmem_wait(vb);
        weigh(vb, 3);
        l += sum[0] + sum[1];
        if ((lo > 0 || hi < kTileT) && (!SHARED || w == 0)) {
          const int u = 2 * (it0 + i - s.i0) + 1;
          if (wait(bars->full + u % p.stages, uint32_t(u / p.stages) & 1u)) {
            if (r < lo || r >= hi) {
              const uint32_t at = smem_u32(ring) + (u % p.stages) * kStage + r * 128;
#pragma unroll
              for (int c = 0; c < NH * 8; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at + (c / 8) * kHalf + (c % 8) * 16), "r"(0) : "memory");
            }
            fence_proxy_async_shared();
          }
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(bars->p_full + w);
      }
      it0 += s.i1 - s.i0;
      // (o, m, l) of the segment
      float* part = tree_part(p, s.pair + int(blockIdx.x));
      if (steps > 0 && wait(bars->o_full + w, (k - 1) & 1u)) tc_fence_after();
      const bool has = steps > 0 && !wait.dead;
      float4* swap = reinterpret_cast<float4*>(qs);  // [D / 4][128]: no score of this segment is still to come
      float f0 = 1.0f, f1 = 0.0f;
      if constexpr (!SHARED) {
        // the second group's part goes to the first through shared memory
        named_barrier(1, 256);
        if (w == 1) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            if (has) {
              tmem_ld32(to + 32 * c, o);
              tmem_wait(o);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              swap[(8 * c + j) * 128 + r] = has ? make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]),
                                                              __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]))
                                                : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
          other[r] = make_float2(m, l);
        }
        named_barrier(1, 256);
        if (w == 0) {
          const float2 ml = other[r];
          const float top = fmaxf(m, ml.x);
          f0 = exp2_from(m, top), f1 = exp2_from(ml.x, top);
          m = top;
          l = fmaf(f1, ml.y, l * f0);
        }
      }
      if (SHARED || w == 0) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (has) {
            tmem_ld32(to + 32 * c, o);
            tmem_wait(o);
          }
          if (x < cols.n) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float4 y = has ? make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]), __uint_as_float(o[4 * j + 2]),
                                           __uint_as_float(o[4 * j + 3]))
                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if constexpr (!SHARED) {
                const float4 z = swap[(8 * c + j) * 128 + r];
                y.x = fmaf(f1, z.x, f0 * y.x), y.y = fmaf(f1, z.y, f0 * y.y);
                y.z = fmaf(f1, z.z, f0 * y.z), y.w = fmaf(f1, z.w, f0 * y.w);
              }
              reinterpret_cast<float4*>(part)[(8 * c + j) * p.RT + x] = y;
            }
          }
        }
        if (x < cols.n) *reinterpret_cast<float2*>(part + p.RT * D + 2 * x) = make_float2(m, l);
      }
      if constexpr (!SHARED) named_barrier(1, 256);  // before the next rows of Q
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

const void* tree_tile_kernel_for(int dtype, int D, bool shared) {
#define SD_TILE(E, DD) \
  return shared ? reinterpret_cast<const void*>(&tree_tile_kernel<E, DD, true>) : reinterpret_cast<const void*>(&tree_tile_kernel<E, DD, false>)
  if (dtype == 1 && D == 64) SD_TILE(__half, 64);
  if (dtype == 1 && D == 128) SD_TILE(__half, 128);
  if (dtype == 2 && D == 64) SD_TILE(__nv_bfloat16, 64);
  if (dtype == 2 && D == 128) SD_TILE(__nv_bfloat16, 128);
#undef SD_TILE
  return nullptr;
}

}  // namespace sd
