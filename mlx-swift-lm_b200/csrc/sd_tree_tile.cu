// sd_tree_tile.cu -- attention of many (node, query head) columns per sequence
// on the fifth-generation tensor cores, for 16-bit pools and for codes of bf16
// ones; compiled once per (SD_E, SD_BITS) pair. See sd_tree.cuh for what it is a
// part of.
//
// A pair's columns are the rows of 128-row accumulators: S = Q K^T (128 rows x
// 64 tokens), P = 2^(S - m), O += P V. S, P -- the second product's left operand --
// and O live in tensor memory, Q, K and V are 128B-swizzled tiles in shared memory
// (TMA, one box per page and 64 dimensions). One warp loads, two groups of four
// warps hold a row per thread and make P, each with its own S and O and a warp that
// issues its products:
//   SHARED: the pair has up to 256 columns, 128 per group, and both groups use
//     every tile;
//   else: it has up to 128, both groups have the same ones, and tiles go to the
//     groups in turn, whose parts are joined at a segment's end.
// P has its place beside S, so that the scores of the next tile are made as
// soon as this one's have been read, and P V while the next is weighed: only the
// store of P waits for the product before.
// P is two values of the element type, a high and a low half, as in the kernel for
// few columns: 16 bits of it (22 of fp16), so that a result has its own rounding and
// nothing else, whatever the number of columns. One half alone was half a step of
// every weight, and a result 1.4 times as far off in the mean square (rows of bf16 up
// to 5e-3 off the rounded exact result, 2e-3 being the tolerance); it took 154 us for
// the largest case below instead of 180, and 38 instead of 40 for one sequence of 32K.
//
// The running maximum lags by up to kSlack, as in a decode; when it moves, its
// group rescales O in tensor memory. The nodes are the sequence's last tokens: a
// row's bits of them and the first token that it sees make 64 bits for a half,
// and scores without theirs are replaced. But 0 * NaN is NaN: rows of V outside
// the range may hold anything and are zeroed in shared memory, and so are
// infinities and not-a-numbers in a node's row, which a row that does see the
// node gets back at the end.
// Bound by the weighing warps and the products: 64 tokens of 256 columns are 16384
// exponentials, 1024 cycles of an SM, and some 1700 cycles of products, and take some
// 2900: each scheduler has two such warps, whose chain (load, maxima, exponentials,
// halves, store, signal) leaves gaps. Measured with the merge, 32 query and 8 kv heads
// of 128 in bf16: 4 sequences of 32K tokens with 64 nodes 180 to 186 us (2.9 TB/s, 0.74 PFLOP/s
// of attention, half as much again with the low halves; 216 us at the 1500 MHz that
// the power limit leaves when it goes on), one with 32 nodes 40 us (3.3 TB/s); 4 x 32K in
// 4 bits with 16 nodes 200 us.
//
// Codes: the loading warp brings them as they are, with their scales; eight more
// make tiles of values of them, s c + b in fp32 and then two bf16 values, a high and a low
// half: 16 bits of a value, and fp32's range, so that a token's size does not matter to
// another's, be it seen or not. The products are q times both halves of K, and three of
// P and V, less the low halves' own. Bound by the converting warps: ten instructions make
// two values, and a tile takes one of their two teams 4500 cycles, 2600 a tile with what they
// wait for (P V first and then the next scores, which wait for the team: the other order
// kept V's place from the team, 291 us instead of 200 for 4 x 32K in 4 bits with 16
// nodes). One fp16 value with a power of two per tile took 126 us there, but it was
// off by 2^-12 of every value, which keys with a large channel make 8e-3 of a result, and
// lost a tile's small values beside a large one that a row need not even see.
#include "sd_tree.cuh"

#if !defined(SD_E) || !defined(SD_BITS)
#error "SD_E and SD_BITS must be defined"
#endif

#if SD_E == 1 && SD_BITS != 0
#error "codes of fp16 pools: tree_attend_kernel"
#elif SD_E == 1
using ET = __half;
#else
using ET = __nv_bfloat16;
#endif

namespace sd {

namespace {

constexpr int kTileT = kTreeTileTokens;
static_assert(kTileT == 64, "a row's bits of a tile are a mask's");
constexpr int kTmemCols = 512;
// Tensor memory columns of the first group's S, its P's high and low halves, and its O; the second's are 128 on.
constexpr int kSCol = 0, kPCol = 64, kOCol = 256;

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
// A whole warp calls these and one thread of it, always the same, issues: what the products' operands are computed
// from stays uniform.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(int(add))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(int(add))
      : "memory");
}
// The barrier gets one arrival when the products issued so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar)
      : "memory");
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
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      SD_W8(v, 0), SD_W8(v, 8), SD_W8(v, 16), SD_W8(v, 24)
      : "memory");
}

// --- waits: bounded; the answer is the warp's, as the tensor memory accesses are ---
// A wait that has to go on is out of line: every instruction in the loops here is fetched again for each tile. (Not in
// the kernel for codes: a call keeps the registers from being shared out anew.)
static __device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, int* flags) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, flags));
}
constexpr uint32_t kMostTries = 3u << 19;  // a try waits for 1.36 us (measured): 2 s; the time read as well cost 4%
template <bool CALL>
struct Waiter {
  int* flags;
  bool dead;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) {
    if constexpr (CALL) {
      if (!dead && !__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) dead = !wait_on(bar, parity, flags);
    } else {
      if (!dead && !__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
        uint32_t tries = 0;
        while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)) && ++tries < kMostTries) {}
        dead = tries == kMostTries;
        if (dead && flags) atomicOr(flags, kErrTimeout);
      }
    }
    return !dead;
  }
};
// One arrival for a warp, after what its lanes did: a barrier takes some three cycles for each, and 128 of them made
// every signal between the warps 430 cycles late.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n @e mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(smem_u32(bar))
               : "memory");
}
// A wait names a phase by its parity: right as long as the phase before it is done and the one after it is not. So
// what goes with P has a barrier per buffer, as the other buffer's may be a phase ahead.

// Two products and sums in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// Whether one of the threads says so: a barrier of n threads.
__device__ __forceinline__ bool barrier_or(int id, int n, bool p) {
  int any;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, %3, p;\n selp.b32 %0, 1, 0, q;\n}\n"
      : "=r"(any) : "r"(int(p)), "r"(id), "r"(n) : "memory");
  return any != 0;
}
// Makes zeros of those of a word's two values that are not finite; true if there was one.
template <typename E>
__device__ __forceinline__ bool finite2(uint32_t& w) {
  constexpr uint32_t top = __is_same(E, __half) ? 0x7c00u : 0x7f80u;
  const bool a = (w & top) == top, b = (w & (top << 16)) == (top << 16);
  if (a) w &= 0xffff0000u;
  if (b) w &= 0x0000ffffu;
  return a || b;
}

// Codes as floats, 2^23 + c less 2^23: two neighbouring bytes of a word, or two nibbles four apart, bits 4 i of each half,
// as 16^i times as much. So the tiles of nibbles hold codes 0 4 1 5 2 6 3 7 of every eight dimensions, as their rows of Q
// do, and O has its columns in that order.
__device__ __forceinline__ float2 bytes2(uint32_t w, int i) {
  return add2(make_float2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7650 + i)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7651 + i))),
              make_float2(-8388608.0f, -8388608.0f));
}
__device__ __forceinline__ float2 nibbles2(uint32_t w, int i) {
  return add2(make_float2(__uint_as_float((w & (15u << (4 * i))) | 0x4B000000u), __uint_as_float((w >> 16 & (15u << (4 * i))) | 0x4B000000u)),
              make_float2(-8388608.0f, -8388608.0f));
}
// Two values' high halves (cut off, so that they are finite where the values are) and low ones.
__device__ __forceinline__ void halves2(float2 x, uint32_t& high, uint32_t& low) {
  const uint32_t a = __float_as_uint(x.x), b = __float_as_uint(x.y);
  high = __byte_perm(a, b, 0x7632);
  const float2 r = fma2(make_float2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)), make_float2(-1.0f, -1.0f), x);
  low = pack2<__nv_bfloat16>(r.x, r.y);
}
// Whether all codes of a group stand for finite values.
template <int BITS>
__device__ __forceinline__ bool finite_group(float scale, float bias) {
  return fabsf(bias) < INFINITY && fabsf(fmaf(scale, float((1 << BITS) - 1), bias)) < INFINITY;
}

struct TileBars {
  uint64_t full[kTreeTileStages], empty[kTreeTileStages];
  uint64_t q_full[2], s_full[2], s_free[2], p_full[2], o_full[2];  // of a group
  uint64_t raw_full[kTreeRawStages], raw_empty[kTreeRawStages];
  uint64_t started, done;
  uint32_t tmem;
};
static_assert(sizeof(TileBars) <= kTreeTileBarBytes, "room in the layout");

}  // namespace

template <typename E, int BITS, int D, bool SHARED>
__global__ void __launch_bounds__(BITS ? kTreeCodeThreads : kTreeTileThreads, 1)
tree_tile_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV) {
  constexpr int NH = D / 64, kQHalf = 128 * 128, kHalf = kTileT * 128;  // bytes of 64 dimensions of Q, of a tile
  constexpr int kQ = NH * kQHalf, kTile = NH * kHalf, kStage = BITS ? 2 * kTile : kTile;  // of codes: high halves, then low ones
  constexpr int kThreads = BITS ? kTreeCodeThreads : kTreeTileThreads;
  static_assert(!BITS || !SHARED, "codes: pairs of up to 128 columns, there is no room for more rows of Q beside the tiles");
  constexpr float kUp = __is_same(E, __half) ? 7.0f : 0.0f;  // as in a decode: fp16 weights up to 2^(kUp + kSlack)
  constexpr int kQs = tree_tile_queries(D, BITS, SHARED);    // copies of Q: one for both groups makes room for the ring
  constexpr int kRow = BITS ? D * BITS / 8 : 1, kSb = BITS ? kTileT * (D / 64) * 2 : 0;  // bytes: a row of codes, a tile's scales
  constexpr int kRaw = tree_raw_stage(D, BITS);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *qs = sm, *ring = sm + kQs * kQ, *raws = sm + p.q_off;
  TileBars* bars = reinterpret_cast<TileBars*>(sm + p.bar_off);
  int* units = reinterpret_cast<int*>(sm + p.prefix_off);
  int *pairs = units + p.B + 1, *tmp = pairs + p.B + 1;
  __shared__ float2 ml_of[2][SHARED ? 1 : 128];
  __shared__ int4 odd_of[2];  // codes: whether a node's V is not finite, by the four warps that made it; of two tiles
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(bars->full + i, BITS ? 4 : 1);
      mbar_init(bars->empty + i, SHARED ? 2 : 1);  // groups that use the tile
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(bars->q_full + w, kQs == 1 && w == 1 ? 8 : 4);
      mbar_init(bars->s_full + w, 1);
      mbar_init(bars->s_free + w, 4);
      mbar_init(bars->o_full + w, 1);
      mbar_init(bars->p_full + w, 4);
    }
    for (int i = 0; i < kTreeRawStages; ++i) {
      mbar_init(bars->raw_full + i, 33);
      mbar_init(bars->raw_empty + i, 4);
    }
    mbar_init(&bars->started, 4);
    mbar_init(&bars->done, 2);
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
  tree_line<kThreads>(p, kTileT, units, pairs, tmp);  // with barriers
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  const Pieces pieces(p, units[p.B]);
  const bool work = int(blockIdx.x) < pieces.n;
  TreeWalk walk(p, units, pairs, work ? pieces.begin(blockIdx.x) : 0, work ? pieces.begin(blockIdx.x + 1) : 0);
  TreeSegment s;
  int it0 = 0;  // tiles of the segments before
  Waiter<BITS == 0> wait{p.flags, false};

  // The registers of a launch for codes (20 warps x 96) shared out anew: 8 x 144 for the weights, 12 x 64.
  if (warp >= 8) {
    if constexpr (BITS) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
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
        const int t0 = sq.begin / kTileT, last_slot = (sq.end - 1) >> p_log, first_slot = sq.begin >> p_log;
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
          const bool need = lane < nb && tj < sq.end && tj + pb > sq.begin;
          int y = oob_row;
          if (need) {
            if (page >= 0 && page < p.n_pages) y = int((int64_t(page) * p.Hkv + s.h) * p.P + (tj & (p.P - 1)));
            else if (p.flags) atomicOr(p.flags, kErrBadIndex);
          }
          const int n_box = __popc(__ballot_sync(0xffffffffu, need));
          if constexpr (BITS) {  // K and V and their scales, as they are, in one stage
            if (use >= p.raw_stages && !wait(bars->raw_empty + st, round ^ 1u)) break;
            uint64_t* full = bars->raw_full + st;
            uint8_t* stage = raws + st * kRaw;
            if (lane == 0) mbar_arrive_expect_tx(full, uint32_t(n_box * 2 * pb * kRow));
            __syncwarp();
            if (need) {
              tma_load_3d(stage + lane * pb * kRow, &tmK, 0, y, 0, full, pol);
              tma_load_3d(stage + (kTileT + lane * pb) * kRow, &tmV, 0, y, 0, full, pol);
            }
            constexpr int ROW = D / 64 * 2, CPA = kSb / 16;  // bytes of a token in each array of scales, 16-byte pieces of a tile
            const uint8_t* src[4] = {static_cast<const uint8_t*>(p.k_scales), static_cast<const uint8_t*>(p.k_biases),
                                     static_cast<const uint8_t*>(p.v_scales), static_cast<const uint8_t*>(p.v_biases)};
            const uint32_t sb = smem_u32(stage + 2 * kTileT * kRow);
            const int byte = lane * 16, j = min(byte / ROW / pb, nb - 1);  // the box this piece's tokens lie in
            const int64_t kr = __shfl_sync(0xffffffffu, y, j);
            const bool good = __shfl_sync(0xffffffffu, int(need && y != oob_row), j);
            if (lane < CPA) {
#pragma unroll
              for (int x = 0; x < 4; ++x)
                cp_async16_zfill(sb + x * kSb + byte, good ? src[x] + (kr * ROW + byte - j * pb * ROW) : src[x], good ? 16 : 0);
            }
            cp_async_arrive(full);
            ++use;
            if (++st == p.raw_stages) {
              st = 0;
              round ^= 1u;
            }
          } else {
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
      }
      if (wait.dead) {  // what is under way lands in this CTA's shared memory
        uint64_t* full = BITS ? bars->raw_full : bars->full;
        const int n = BITS ? p.raw_stages : p.stages;
        for (int u = max(0, use - n); u < use; ++u) mbar_wait(full + u % n, uint32_t(u / n) & 1u, nullptr);
      }
    } else if (warp == 9 || warp == 10) {  // ---- products of a group ----
      const int w = warp - 9;
      uint32_t seg = 0, k = 0;  // segments that the group took part in and tiles: the parities of its barriers
      const uint64_t q = operand_desc(0, 16, 1024) + ((smem_u32(qs) + (kQs == 2 ? w * kQ : 0)) >> 4);
      const uint64_t kd0 = operand_desc(0, 16, 1024) + (smem_u32(ring) >> 4), vd0 = operand_desc(0, kHalf, 1024) + (smem_u32(ring) >> 4);
      const uint32_t ds = tmem + kSCol + w * 128, dp = tmem + kPCol + w * 128, dO = tmem + kOCol + w * 128;
      const uint32_t empty = smem_u32(bars->empty), o_full = smem_u32(bars->o_full + w), s_full = smem_u32(bars->s_full + w);
      while (walk.next(s)) {
        const int nt = s.i1 - s.i0, n = SHARED ? nt : (nt + 1 - w) / 2;
        if (n > 0) {
          // A group without tiles (a segment of one) loads no rows of Q: it could run ahead by more than a phase. The
          // second group begins when the first has weighed its first tile: out of step, one's exponentials overlap the
          // other's loads, maxima and stores.
          if (w == 1 && k == 0) wait(&bars->started, 0);
          wait(bars->q_full + w, seg++ & 1u);
        }
        const int u = 2 * (it0 + (SHARED ? 0 : w));
        int ks = u % p.stages, kp = (u / p.stages) & 1, vs = (u + 1) % p.stages, vp = ((u + 1) / p.stages) & 1;
        // The scores of tile i + 1, then P V of tile i. The first scores follow the rows of Q: with those the group has
        // read what it needs of its last S and O. Codes: P V of tile i before the scores of the next one, whose keys' place
        // is made free by this one's scores and its values' by this P V.
#pragma unroll 1
        for (int i = BITS ? 0 : -1; i < n && !wait.dead; ++i) {
          const int next = BITS ? i : i + 1;
          if (next < n) {
            if (!wait(bars->full + ks, uint32_t(kp)) || (next > 0 && !wait(bars->s_free + w, (k + next - 1) & 1u))) break;
            tc_fence_after();
            const uint64_t kd = kd0 + ks * (kStage >> 4);
#pragma unroll
            for (int c = 0; c < kStage / kTile * (D / 16); ++c) {  // codes: K's high halves, then the low ones
              const int cc = c % (D / 16);
              mma_ss(ds, q + (cc / 4) * (kQHalf >> 4) + (cc % 4) * 2,
                     kd + c / (D / 16) * (kTile >> 4) + (cc / 4) * (kHalf >> 4) + (cc % 4) * 2, product_desc<E>(kTileT, false), c > 0);
            }
            mma_commit(s_full);
            mma_commit(empty + ks * 8);
            ks += SHARED ? 2 : 4;
            if (ks >= p.stages) ks -= p.stages, kp ^= 1;
          }
          if (i >= 0) {
            if (!wait(bars->full + vs, uint32_t(vp)) || !wait(bars->p_full + w, (k + i) & 1u)) break;
            tc_fence_after();
            const uint64_t v = vd0 + vs * (kStage >> 4);
#pragma unroll
            for (int c = 0; c < kTileT / 8; ++c)  // P's high half, then its low one
              mma_ts(dO, dp + c * 8, v + c % (kTileT / 16) * (2048 >> 4), product_desc<E>(D, true), i > 0 || c > 0);
            if constexpr (BITS != 0) {  // the high half with V's low one
#pragma unroll
              for (int c = 0; c < kTileT / 16; ++c) mma_ts(dO, dp + c * 8, v + (kTile >> 4) + c * (2048 >> 4), product_desc<E>(D, true), true);
            }
            mma_commit(o_full);
            mma_commit(empty + vs * 8);
            vs += SHARED ? 2 : 4;
            if (vs >= p.stages) vs -= p.stages, vp ^= 1;
          }
        }
        k += n;
        it0 += nt;
      }
      mma_commit(smem_u32(&bars->done));  // no product may read shared memory that is no longer this CTA's
      mbar_wait(&bars->done, 0, p.flags);
    } else if (BITS && warp >= 12) {  // ---- codes into tiles of halves ----
      if constexpr (BITS) {
        constexpr int NG = D / 64, EPC = 128 / BITS, CPR = kRow / 16;  // groups, codes of 16 bytes, such pieces of a row
        // Four warps for every other tile: what a tile waits for (codes, a free stage) is hidden by the other four's.
        // The numbers of stages are such that a stage stays with one of these teams.
        const int team = (warp - 12) >> 2, ct = tid & 127;
        constexpr int PH = 64 / EPC;  // pieces of 64 dimensions: eight lanes have those of neighbouring rows, and what they
                                      // store at a time lies in eight different 16-byte columns
        int rs = team, ks = 2 * team;  // the tile's stages: of codes, of K (V's is the next one); their phases
        uint32_t rp = 0, kp = 0;
        while (walk.next(s)) {
          const TreeSeq sq = tree_seq(p, s.b);
          const int t0 = sq.begin / kTileT;
          for (int i = s.i0; i < s.i1; ++i, ++it0) {
            if ((it0 & 1) != team) continue;
            const int tok = (t0 + i) * kTileT, lo = sq.begin - tok, hi = sq.end - tok, old = sq.held - tok;
            wait(bars->raw_full + rs, rp);
            const uint8_t* raw = raws + rs * kRaw;
            const uint16_t* small = reinterpret_cast<const uint16_t*>(raw + 2 * kTileT * kRow);  // [K scales, K biases, V ..][64][NG]
#pragma unroll 1
            for (int v = 0; v < 2; ++v) {
              const int st = ks + v;
              wait(bars->empty + st, kp ^ 1u);  // in the first phase at once
              if (!wait.dead) {
                const uint32_t dst = smem_u32(ring) + st * kStage;
                bool odd = false;
#pragma unroll 1
                for (int e = 0; e < kTileT * CPR / 128; ++e) {
                  const int x = ct + 128 * e;
                  const int row = x / (8 * NG) * (8 / PH) + x / PH % (8 / PH), half = x / 8 % NG, c = half * PH + x % PH;
                  const uint4 w = lds128(smem_u32(raw) + (v * kTileT + row) * kRow + c * 16);
                  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                  float sc = __uint_as_float(uint32_t(small[v * 2 * kTileT * NG + row * NG + half]) << 16);
                  float bi = __uint_as_float(uint32_t(small[(v * 2 + 1) * kTileT * NG + row * NG + half]) << 16);
                  if (v && (row < lo || row >= hi)) sc = bi = 0.0f;  // rows that no row sees may hold anything, and 0 * NaN is NaN
                  const bool fine = finite_group<BITS>(sc, bi), node = v && row >= old;
                  odd |= node && !fine;
                  const float2 b2 = make_float2(bi, bi);
#pragma unroll
                  for (int j = 0; j < EPC / 8; ++j) {  // 16 bytes of the tile, and of the low halves'
                    float2 f[4];
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                      const float unit = BITS == 8 ? sc : sc * (1.0f / float(1 << (4 * i4)));
                      const float2 code = BITS == 8 ? bytes2(words[(2 * j + i4 / 2) & 3], 2 * (i4 & 1)) : nibbles2(words[j & 3], i4);
                      f[i4] = fma2(code, make_float2(unit, unit), b2);
                    }
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) halves2(f[i4], h[i4], l[i4]);
                    const int ch = c * EPC / 8 + j;
                    const uint32_t to = dst + (ch / 8) * kHalf + row * 128 + (((ch % 8) ^ (row & 7)) << 4);
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to + kTile), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]) : "memory");
                  }
                  if (!fine) {  // no low halves, which are infinities less themselves, and of a node what is finite: rows that
                                // see it get the rest back
#pragma unroll 1
                    for (int j = 0; j < EPC / 8; ++j) {
                      const int ch = c * EPC / 8 + j;
                      const uint32_t to = dst + (ch / 8) * kHalf + row * 128 + (((ch % 8) ^ (row & 7)) << 4);
                      uint4 h = lds128(to);
                      if (node) finite2<E>(h.x), finite2<E>(h.y), finite2<E>(h.z), finite2<E>(h.w);
                      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(h.x), "r"(h.y), "r"(h.z), "r"(h.w) : "memory");
                      asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to + kTile), "r"(0) : "memory");
                    }
                  }
                }
                if (v) {
                  odd = __any_sync(0xffffffffu, odd);
                  if (lane == 0) reinterpret_cast<int*>(odd_of + team)[warp & 3] = int(odd);
                }
                fence_proxy_async_shared();
                warp_arrive(bars->full + st);
                if (v) warp_arrive(bars->raw_empty + rs);
              }
            }
            if ((rs += 2) >= p.raw_stages) rs -= p.raw_stages, rp ^= 1u;
            if ((ks += 4) >= p.stages) ks -= p.stages, kp ^= 1u;
          }
        }
      }
    }
  } else {  // ---- weights: a row per thread ----
    if constexpr (BITS) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    const int w = warp >> 2, r = tid & 127;  // group, row in it
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // the 32 lanes of tensor memory that this warp reaches
    const uint32_t ts = tmem + lanes + kSCol + w * 128, tp = tmem + lanes + kPCol + w * 128, to = tmem + lanes + kOCol + w * 128;
    const bool neg = p.scale_log2 < 0.0f;
    const float scale = fmaxf(fabsf(p.scale_log2), 1.1754944e-38f);  // -inf times it stays -inf
    uint32_t k = 0;  // tiles of this group
    while (walk.next(s)) {
      const TreeSeq sq = tree_seq(p, s.b);
      const NodeCols cols(p, sq, s.h, s.c);
      const int x = SHARED ? w * 128 + r : r;  // column of the pair
      const int t0 = sq.begin / kTileT;
      if (SHARED || s.i0 + w < s.i1) {  // Q: a thread has one 16-byte chunk of every eighth (or sixteenth) row
        constexpr int CPR = D / 8, RPT = 128 / CPR, N = 128 / RPT;
        const uint32_t q = smem_u32(qs) + (kQs == 2 ? w * kQ : 0);
        const int ch = r % CPR;
        uint4 v[N];
        if (kQs == 2 || w == 0) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int xx = (SHARED ? w * 128 : 0) + r / CPR + RPT * i;
            v[i] = make_uint4(0, 0, 0, 0);
            if (xx < cols.n) v[i] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const E*>(p.q) + cols.row(xx) * D) + ch);
          }
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int row = r / CPR + RPT * i;
            if constexpr (BITS == 4)  // in the order of the codes
              v[i] = make_uint4(__byte_perm(v[i].x, v[i].z, 0x5410), __byte_perm(v[i].x, v[i].z, 0x7632),
                                __byte_perm(v[i].y, v[i].w, 0x5410), __byte_perm(v[i].y, v[i].w, 0x7632));
            const uint32_t at = q + (ch / 8) * kQHalf + row * 128 + (((ch % 8) ^ (row & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[i].x), "r"(v[i].y), "r"(v[i].z), "r"(v[i].w) : "memory");
          }
        }
        fence_proxy_async_shared();
        tc_fence_before();
        warp_arrive(bars->q_full + w);
        if (kQs == 1 && w == 0 && s.i1 - s.i0 > 1) warp_arrive(bars->q_full + 1);  // these rows are the second group's, too
      }
      const int low = x < cols.n ? tree_low(p, sq, cols.node(x)) : 0;
      const uint64_t seen = x < cols.n ? tree_seen(p, sq, cols.node(x)) : 0;
      const int edge = __reduce_max_sync(0xffffffffu, low);
      float m = -INFINITY, l = 0.0f;
      int steps = 0;
      bool odd = false;  // a node has a value that is not finite
      const int n = SHARED ? s.i1 - s.i0 : (s.i1 - s.i0 + 1 - w) / 2;
      const int u0 = 2 * (it0 + (SHARED ? 0 : w)) + 1;
      int vs = u0 % p.stages;  // of the tile's V
      uint32_t vp = uint32_t(u0 / p.stages) & 1u;
#pragma unroll 1
      for (; steps < n; ++steps, ++k) {
        const int tile = SHARED ? steps : 2 * steps + w;  // of the segment
        const int tok = (t0 + s.i0 + tile) * kTileT, lo = sq.begin - tok, hi = sq.end - tok;
        const int old = sq.held - tok;  // rows of the tile before the nodes'
        const bool ends = lo > 0 || old < kTileT;
        // Every group that uses the tile waits for its rows, dead or not; the second one before its own scores, which may
        // wait for the first.
        if (!BITS && SHARED && ends && w == 1) odd |= barrier_or(1, 256, false);
        const bool here = wait(bars->s_full + w, k & 1u);
        if (!BITS && ends && (!SHARED || w == 0)) {
          bool mine = false;
          if (here && wait(bars->full + vs, vp)) {
            const int row = r >> 1;  // a thread has half of it
            const uint32_t at = smem_u32(ring) + vs * kStage + row * 128;
            if (row < lo || row >= old) {
#pragma unroll 2
              for (int c = 0; c < NH * 4; ++c) {
                const int cc = (r & 1) * NH * 4 + c;
                const uint32_t a = at + (cc / 8) * kHalf + (cc % 8) * 16;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row >= old && row < hi) v = lds128(a);
                mine |= finite2<E>(v.x) | finite2<E>(v.y) | finite2<E>(v.z) | finite2<E>(v.w);
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
              }
            }
            fence_proxy_async_shared();
          }
          odd |= SHARED ? barrier_or(1, 256, mine) : barrier_or(2 + w, 128, mine);
        }
        if (!here) continue;
        tc_fence_after();
        if (BITS && old < kTileT && wait(bars->full + vs, vp)) {  // its stage stays until this group's P is used
          const int4 f = odd_of[(it0 + tile) & 1];
          odd |= (f.x | f.y | f.z | f.w) != 0;
        }
        vs += SHARED ? 2 : 4;
        if (vs >= p.stages) vs -= p.stages, vp ^= 1u;
        uint32_t va[32], vb[32];
        tmem_ld32(ts, va);
        tmem_ld32(ts + 32, vb);
        tmem_wait(va);
        tmem_wait(vb);
        tc_fence_before();
        warp_arrive(bars->s_free + w);
        if (neg) {
#pragma unroll
          for (int j = 0; j < 32; ++j) va[j] ^= 0x80000000u, vb[j] ^= 0x80000000u;
        }
        if (ends || tok < edge) {  // some are not seen
          auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };  // the first n rows
          const uint64_t nodes = old >= 64 || old <= -64 ? 0 : old >= 0 ? seen << old : seen >> -old;
          const uint64_t vis = (below(old) & ~below(max(lo, low - tok))) | nodes;
          const uint32_t v0 = uint32_t(vis), v1 = uint32_t(vis >> 32);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            va[j] = v0 & (1u << j) ? va[j] : 0xff800000u;
            vb[j] = v1 & (1u << j) ? vb[j] : 0xff800000u;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 32; j += 4) {  // maxima of three
          mx[0] = fmaxf(fmaxf(mx[0], __uint_as_float(va[j])), __uint_as_float(va[j + 1]));
          mx[1] = fmaxf(fmaxf(mx[1], __uint_as_float(va[j + 2])), __uint_as_float(va[j + 3]));
          mx[2] = fmaxf(fmaxf(mx[2], __uint_as_float(vb[j])), __uint_as_float(vb[j + 1]));
          mx[3] = fmaxf(fmaxf(mx[3], __uint_as_float(vb[j + 2])), __uint_as_float(vb[j + 3]));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
        if (steps == 0) {
          m = top - kUp;
        } else if (__any_sync(0xffffffffu, top > m + (kSlack + kUp))) {
          const float fac = raise_max(m, top - kUp);
          l *= fac;
          if (wait(bars->o_full + w, (k - 1) & 1u)) {  // the last product
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(to + 32 * c, o);
              tmem_wait(o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * fac);
              tmem_st32(to + 32 * c, o);
            }
          }
        }
        const float2 mm = m == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-m, -m), sc2 = make_float2(scale, scale);
        float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
        uint32_t high[32], low2[32];
        auto weigh = [&](const uint32_t (&v)[32], int c) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float2 e = fma2(make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), sc2, mm);
            e.x = ex2(e.x), e.y = ex2(e.y);
            sum[j & 1] = add2(sum[j & 1], e);
            split2<E>(e.x, e.y, high[16 * c + j], low2[16 * c + j]);
          }
        };
        weigh(va, 0);
        weigh(vb, 1);
        if (k > 0 && wait(bars->o_full + w, (k - 1) & 1u)) tc_fence_after();  // what was there has been multiplied
        tmem_st32(tp, high);
        tmem_st32(tp + kTileT / 2, low2);
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tc_wait_st();
        tc_fence_before();
        warp_arrive(bars->p_full + w);
        if (w == 0 && k == 0) warp_arrive(&bars->started);
      }
      it0 += s.i1 - s.i0;
      // (o, m, l) of the segment
      float* part = tree_part(p, s.pair + int(blockIdx.x));
      if (steps > 0 && wait(bars->o_full + w, (k - 1) & 1u)) tc_fence_after();
      const bool has = steps > 0 && !wait.dead;
      // A node's value that is not finite counts in the rows that see it.
      auto add_odd = [&](int c, uint32_t (&o)[32]) {
#pragma unroll 1
        for (uint64_t left = x < cols.n ? seen : 0; left; left &= left - 1) {
          const int t = sq.held + __ffsll(left) - 1, page = __ldcg(p.tables + int64_t(s.b) * p.W + t / p.P);
          if (page < 0 || page >= p.n_pages) continue;
          const int64_t row = (int64_t(page) * p.Hkv + s.h) * p.P + (t & (p.P - 1));
          if constexpr (BITS == 0) {
            const uint32_t* v = reinterpret_cast<const uint32_t*>(p.v_data) + row * (D / 2) + 16 * c;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float f[2];
              unpack_word<E>(__ldcg(v + j), f);
              if (!(fabsf(f[0]) < INFINITY)) o[2 * j] = __float_as_uint(__uint_as_float(o[2 * j]) + f[0]);
              if (!(fabsf(f[1]) < INFINITY)) o[2 * j + 1] = __float_as_uint(__uint_as_float(o[2 * j + 1]) + f[1]);
            }
          } else {
            const int64_t g = row * (D / 64) + c / 2;
            const float sc = Elt<E>::to_f32(static_cast<const E*>(p.v_scales)[g]), bi = Elt<E>::to_f32(static_cast<const E*>(p.v_biases)[g]);
            if (finite_group<BITS>(sc, bi)) continue;
            const uint32_t* v = reinterpret_cast<const uint32_t*>(p.v_data + row * kRow) + c * BITS;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const uint32_t code = __ldcg(v + j * BITS / 32) >> (j * BITS % 32) & ((1u << BITS) - 1);
              const float x = fmaf(float(code), sc, bi);
              if (!(fabsf(x) < INFINITY)) o[j] = __float_as_uint(__uint_as_float(o[j]) + x);
            }
          }
        }
      };
      auto load = [&](int c, uint32_t (&o)[32]) {  // dimensions 32 c ..
        if (has) {
          tmem_ld32(to + 32 * c, o);
          tmem_wait(o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0;
        }
        if constexpr (BITS == 4) {  // out of the order of the codes
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            const uint32_t a = o[j + 1], b = o[j + 2], c = o[j + 3], d = o[j + 4], e = o[j + 5], f = o[j + 6];
            o[j + 4] = a, o[j + 1] = b, o[j + 5] = c, o[j + 2] = d, o[j + 6] = e, o[j + 3] = f;
          }
        }
        if (odd) add_odd(c, o);
      };
      if constexpr (SHARED) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          load(c, o);
          if (x < cols.n) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              reinterpret_cast<uint4*>(part)[(8 * c + j) * 256 + x] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        }
      } else {
        // each group finishes half of the dimensions and hands the other half over, 32 at a time, in the place of Q: no
        // score of this segment is still to come
        uint4* swap = reinterpret_cast<uint4*>(qs) + w * 8 * 128;  // [8][128]
        const uint4* from = reinterpret_cast<const uint4*>(qs) + (1 - w) * 8 * 128;
        ml_of[w][r] = make_float2(m, l);
        float most = 0.0f, f0 = 0.0f, f1 = 0.0f;
        float2 ml;
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t o[32];
          named_barrier(1, 256);  // Q, or what was handed over before, has been read
          load((1 - w) * (D / 64) + c, o);
#pragma unroll
          for (int j = 0; j < 8; ++j) swap[j * 128 + r] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          named_barrier(1, 256);
          ml = ml_of[1 - w][r];
          most = fmaxf(m, ml.x), f0 = exp2_from(m, most), f1 = exp2_from(ml.x, most);
          load(w * (D / 64) + c, o);
          if (x < cols.n) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint4 z = from[j * 128 + r];
              auto join = [&](uint32_t a, uint32_t b) { return fmaf(f1, __uint_as_float(b), f0 * __uint_as_float(a)); };
              reinterpret_cast<float4*>(part)[(w * (D / 8) + 8 * c + j) * 128 + x] =
                  make_float4(join(o[4 * j], z.x), join(o[4 * j + 1], z.y), join(o[4 * j + 2], z.z), join(o[4 * j + 3], z.w));
            }
          }
        }
        m = most;
        l = w == 0 ? fmaf(f1, ml.y, l * f0) : fmaf(f0, l, ml.y * f1);
        named_barrier(1, 256);  // before the next rows of Q
      }
      if (x < cols.n && (SHARED || w == 0)) *reinterpret_cast<float2*>(part + p.RT * D + 2 * x) = make_float2(m, l);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

#define SD_NAME2(e, b) tree_tile_e##e##_b##b
#define SD_NAME(e, b) SD_NAME2(e, b)
const void* SD_NAME(SD_E, SD_BITS)(int D, bool shared) {
#if SD_BITS == 0
  if (shared) return D == 64 ? reinterpret_cast<const void*>(&tree_tile_kernel<ET, 0, 64, true>)
                             : reinterpret_cast<const void*>(&tree_tile_kernel<ET, 0, 128, true>);
#endif
  return D == 64 ? reinterpret_cast<const void*>(&tree_tile_kernel<ET, SD_BITS, 64, false>)
                 : reinterpret_cast<const void*>(&tree_tile_kernel<ET, SD_BITS, 128, false>);
}

}  // namespace sd
