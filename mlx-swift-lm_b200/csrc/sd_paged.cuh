// sd_paged.cuh -- attention of one new token per sequence over a paged KV pool.
//
// out[b, hq] = sum_t e^(s_t) v_t / (sum_t e^(s_t) + e^(sink)), s_t = scale q.k_t,
// over the tokens t in [max(0, len - window), len) of sequence b, whose keys
// and values lie in the pages that row b of the table names; an empty range
// gives zeros.
//
// The call reads every K and V byte once and computes 2 * G products per
// element: it is bound by HBM, and the design keeps HBM busy whatever the
// batch looks like. The tokens are cut into tiles (PagedFmt::kTile); the tiles
// of all (sequence, kv head) pairs, in order, are one line that is cut into
// equal pieces, one per CTA (two CTAs per SM, all resident). A CTA walks its
// piece: one producer warp streams the tiles into a ring of stages (TMA for K
// and V, cp.async for scales and biases) and four warps attend, each to its
// own quarter of every tile with its own running (m, l, o) -- no barrier
// between warps until a segment (the CTA's share of one pair) ends. A segment
// that is a whole pair is written out; the others leave (m, l, o) in the
// workspace and paged_merge_kernel joins them in CTA order, so results do not
// depend on timing (the last bits of a sequence do depend on the other lengths
// of the batch, which say where it is cut). The lengths are read on the device
// only, so a captured graph serves growing sequences.
//
// The products have at most 16 query heads on one side, so they run on
// register-level mma (16-bit rows and codes) or FMA (fp32), not on tcgen05
// tiles, whose M of 64 or more would be mostly padding. Measured, 32 query and
// 8 kv heads of 128, inputs beyond L2: 16 ragged bf16 sequences of up to 128K
// tokens (4.2 GB) 609 us, 6.9 TB/s; 4 x 128K in 8 bits (1.1 GB) 182 us, 6.3
// TB/s; the same in 4 bits (0.6 GB) 152 us, 4.0 TB/s, bound by the latency of a
// tile's chain of instructions (56% of the issue slots used); 4 x 32K in fp32
// (1.1 GB) 175 us, 6.1 TB/s; one bf16 sequence of 32K (134 MB) 27 us, of which
// 20 are the bytes and the rest start (first tile 3 us after the launch) and
// merge (2.5 us).
//
// The running maximum m is a lower bound of the true one by at most kSlack
// (log2 units): it moves, and l and o are rescaled, only when a score passes
// m + kSlack, which one vote per tile finds; p stays below 2^kSlack (for dense
// fp16 m stands lower still, see there).
#pragma once

#include "sd_device.cuh"
#include "sd_paged.h"

namespace sd {

constexpr float kSlack = 8.0f;

// c += A(16x16, row-major) * B(16x8, col-major), all four A registers.
template <typename E>
__device__ __forceinline__ void mma_full(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (sizeof(E) == 2 && !__is_same(E, __half)) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    mma16816_f16(c, a0, a1, a2, a3, b0, b1);
  }
}

// 16-byte cp.async that fills with zeros when `bytes` is 0.
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// The barrier counts one arrival of this thread when its cp.asyncs so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Where a tile's rows lie in its stage: boxes of PB rows, each [kNBox][PB][kBoxBytes] swizzled by TMA.
template <class F>
struct TileAddr {
  uint32_t base;  // shared address of the K (or V) part
  int pb_log;     // log2 of the rows per box
  // First byte of row `row` of the box columns.
  __device__ __forceinline__ uint32_t row_at(int row) const {
    return base + uint32_t(((row >> pb_log) << pb_log) * F::kRowBytes + (row & ((1 << pb_log) - 1)) * F::kBoxBytes);
  }
};
// What a lane's ldmatrix address adds to row_at of its 16 rows, for row `r`
// of them (boxes hold 16 rows at least) and chunk 2c + odd: the swizzle of a
// row does not depend on which 16 rows it is in, and an even chunk number
// joins the odd bit by xor.
template <class F>
struct LaneAddr {
  uint32_t off, x;
  __device__ __forceinline__ LaneAddr(int r, int odd) {
    off = uint32_t(r * F::kBoxBytes);
    x = (((off >> 7) & (F::kCpb - 1u)) << 4) ^ uint32_t(odd * 16);
  }
  __device__ __forceinline__ uint32_t at(uint32_t rows, int chunk, int pb_log) const {  // chunk: even
    return rows + off + uint32_t((chunk / F::kCpb) << pb_log) * F::kBoxBytes + (x ^ uint32_t((chunk % F::kCpb) * 16));
  }
};

struct TileView {
  const uint8_t* stage;
  int pb_log;
  int lo, hi;  // valid token rows of the tile
};

// (m, l) and o of one warp in the combine buffer.
template <int D>
struct WarpPart {
  float *o, *ml;
  __device__ __forceinline__ WarpPart(float* buf, int G, int warp) {
    o = buf + warp * paged_warp_floats(G, D);
    ml = o + G * (D + 4);
  }
};

// 2^x by the hardware's instruction (relative error 2^-22; results below
// 2^-126 are zero, which a softmax weight may be).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_from(float s, float m) { return ex2(s - (m == -INFINITY ? 0.0f : m)); }

// New running maximum and the factor for what was summed under the old one.
__device__ __forceinline__ float raise_max(float& m, float mx) {
  const float mn = fmaxf(m, mx);
  const float f = mn == -INFINITY ? 1.0f : ex2(m - mn);
  m = mn;
  return f;
}

// ---------------------------------------------------------------------------
// 16-bit K and V on the tensor cores (bound by HBM: issue slots are 21% used),
// tokens as the rows of the tile:
// S^T = K q^T (m16n8k16: 16 tokens x 8 heads), O^T = V^T P^T (16 dims x 8
// heads). G <= 8 heads fill the 8 columns of one block, up to 16 two blocks.
// Lane (g, tq) = (lane / 4, lane % 4): S^T rows g, g + 8 are tokens and its
// columns 2tq, 2tq + 1 heads, the same heads as in O^T, so the softmax state
// of a head lies where its outputs are. P^T gets its operand layout from
// movmatrix. p is used as hi + lo halves of the element type (about 16 bits
// of it for bf16): a single bf16 p would cost as much accuracy as the final
// rounding does, and the extra mma is free next to the loads. fp16 has no
// halves below 2^-24, so there m stands 2^kUp below the maximum: p goes up to
// 2^(kUp + kSlack) = 2^15, and a weight keeps its bits down to 2^-(24 + kUp) of
// the maximum's. At a kUp of 0 the many small weights beside an attention sink
// (each below 2^-25) were lost to o, though not to l.
// ---------------------------------------------------------------------------
template <typename E, int D, int NB>
struct DenseAttend {
  using F = PagedFmt<2, 0, D>;
  static constexpr int NC = D / 16;
  static constexpr float kUp = __is_same(E, __half) ? 7.0f : 0.0f;
  uint32_t qb[NB][NC][2];
  float m[NB][2], l[NB][2], o[NB][NC][4];

  __device__ __forceinline__ void begin(const PagedParams& p, const float*, int b, int h, int, int lane) {
    const int g = lane >> 2, tq = lane & 3;
    const uint32_t* q = static_cast<const uint32_t*>(p.q);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int hd = 8 * nb + g;
      const int64_t row = (int64_t(b) * p.Hkv * p.G + int64_t(h) * p.G + hd) * (D / 2);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        qb[nb][c][0] = hd < p.G ? q[row + 8 * c + tq] : 0u;
        qb[nb][c][1] = hd < p.G ? q[row + 8 * c + 4 + tq] : 0u;
        o[nb][c][0] = o[nb][c][1] = o[nb][c][2] = o[nb][c][3] = 0.0f;
      }
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.0f;
    }
  }

  __device__ __forceinline__ void tile(const PagedParams& p, const float*, const TileView& t, int warp, int lane) {
    constexpr int TW = F::kTile / kPagedWarps;
    static_assert(TW == 16, "one m-tile per warp");
    const int g = lane >> 2, tq = lane & 3, mq = lane >> 3, r8 = lane & 7;
    const int r0 = warp * TW;
    const int lo = t.lo - r0, hi = t.hi - r0;  // valid rows of this warp's 16
    if (hi <= 0 || lo >= TW) return;
    const uint32_t krows = TileAddr<F>{smem_u32(t.stage), t.pb_log}.row_at(r0), vrows = krows + F::kKvBytes;
    const LaneAddr<F> ka(8 * (mq & 1) + r8, mq >> 1), va(8 * (mq >> 1) + r8, mq & 1);
    float acc[2][NB][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) acc[i][nb][0] = acc[i][nb][1] = acc[i][nb][2] = acc[i][nb][3] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t a0, a1, a2, a3;
      ldsm_x4(ka.at(krows, 2 * c, t.pb_log), a0, a1, a2, a3);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) mma_full<E>(acc[c & 1][nb], a0, a1, a2, a3, qb[nb][c][0], qb[nb][c][1]);
    }
    const bool ok0 = g >= lo && g < hi, ok1 = g + 8 >= lo && g + 8 < hi;
    float s[NB][4];
    bool up = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = (acc[0][nb][i] + acc[1][nb][i]) * p.scale_log2;
        s[nb][i] = (i < 2 ? ok0 : ok1) ? v : -INFINITY;
        up |= s[nb][i] > m[nb][i & 1] + (kSlack + kUp);
      }
    }
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(s[nb][e], s[nb][2 + e]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float f = raise_max(m[nb][e], mx - kUp);
          l[nb][e] *= f;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            o[nb][c][e] *= f;
            o[nb][c][2 + e] *= f;
          }
        }
      }
    }
    uint32_t ph[NB][2], pl[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[nb][i] = exp2_from(s[nb][i], m[nb][i & 1]);
        l[nb][i & 1] += s[nb][i];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t hi2, lo2;
        split2<E>(s[nb][2 * e], s[nb][2 * e + 1], hi2, lo2);
        ph[nb][e] = movm_trans(hi2);
        pl[nb][e] = movm_trans(lo2);
      }
    }
    const bool whole = lo <= 0 && hi >= TW;
    // tokens 2tq, 2tq + 1 (m0) and 2tq + 8, 2tq + 9 (m1) of the V fragments: rows outside [lo, hi) may hold
    // anything, not-a-numbers included, and 0 * NaN is NaN
    auto keep = [&](int tk) { return (tk >= lo && tk < hi ? 0xffffu : 0u) | (tk + 1 >= lo && tk + 1 < hi ? 0xffff0000u : 0u); };
    const uint32_t m0 = keep(2 * tq), m1 = keep(2 * tq + 8);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t a0, a1, a2, a3;
      ldsm_x4_t(va.at(vrows, 2 * c, t.pb_log), a0, a1, a2, a3);
      if (!whole) {
        a0 &= m0;
        a1 &= m0;
        a2 &= m1;
        a3 &= m1;
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        mma_full<E>(o[nb][c], a0, a1, a2, a3, ph[nb][0], ph[nb][1]);
        mma_full<E>(o[nb][c], a0, a1, a2, a3, pl[nb][0], pl[nb][1]);
      }
    }
  }

  __device__ __forceinline__ void end(const PagedParams& p, const WarpPart<D>& w, int lane) {
    const int g = lane >> 2, tq = lane & 3;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float ls = l[nb][e];
        ls += __shfl_xor_sync(0xffffffffu, ls, 4);
        ls += __shfl_xor_sync(0xffffffffu, ls, 8);
        ls += __shfl_xor_sync(0xffffffffu, ls, 16);
        const int hd = 8 * nb + 2 * tq + e;
        if (hd < p.G) {
          if (g == 0) {
            w.ml[2 * hd] = m[nb][e];
            w.ml[2 * hd + 1] = ls;
          }
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            w.o[hd * (D + 4) + 16 * c + g] = o[nb][c][e];
            w.o[hd * (D + 4) + 16 * c + 8 + g] = o[nb][c][2 + e];
          }
        }
      }
    }
  }
};

// Codes as fp16 without removing the offset: two bytes of r as 1024 + c (sel
// takes the low halves' bytes from r, the high ones, 0x64, from byte 1 of
// `magic`); or the nibbles at bits [4 hi, 4 hi + 4) of r's halves as 1024 + c
// (1024 + 16 c for hi). magic is 0x64006400, fp16 1024 twice, as a kernel
// argument: as a literal it would make two instructions of each of these.
__device__ __forceinline__ uint32_t raw_u8(uint32_t r, uint32_t sel, uint32_t magic) { return __byte_perm(r, magic, sel); }
__device__ __forceinline__ uint32_t raw_u4(uint32_t r, int hi, uint32_t magic) {
  return (r & (hi ? 0x00F000F0u : 0x000F000Fu)) | magic;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Scales (or biases) of token t for every group, in fp32, from shared memory.
template <typename E, int NG>
__device__ __forceinline__ void load_groups(uint32_t a, int t, float (&f)[NG]) {
  if constexpr (sizeof(E) == 4 && NG == 2) {
    const uint2 w = lds64(a + 8 * t);
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y);
  } else if constexpr (sizeof(E) == 4) {
    f[0] = __uint_as_float(lds32(a + 4 * t));
  } else if constexpr (NG == 2) {
    unpack_word<E>(lds32(a + 4 * t), f);
  } else {
    uint16_t w;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(a + 2 * t));
    f[0] = Elt<E>::to_f32(__builtin_bit_cast(E, w));
  }
}

// ---------------------------------------------------------------------------
// 4/8-bit codes, the same products, with the codes as exact fp16 integers.
// The chain of instructions bounds this path as much as bytes do, so the
// conversion is short: one byte permute (or mask) puts codes into the mantissas of 1024 + c,
// or 1024 + 16 c for the nibbles that lie 4 bits higher.
//   q.k = s_k (q.c) + b_k sum(q)  per 64-dim group, in fp32. bf16 pools leave
// the offset in where it is at most four times the codes' range -- 1024 for 8
// bits, 1024 / 16 = 64 for a nibble whose place counts 16: the accumulator
// starts at -1024 sum(q') (q' = q in fp16, a 16th of it at those places). That
// costs fp32 3 bits at most; a score is off by at most 2^-20 (four mma, two
// units of the largest partial sum each) of scale s_k sum((c + offset) |q|) per
// group. The low nibble's 1024 would be 68 times the range, 6 bits, and scores
// of wide keys (a range of 240) under queries of one sign off by up to 3e-2, so
// it is subtracted there (4 x 128K tokens 148.6 -> 151.6 us), as it is in fp16
// and fp32 pools throughout. fp32 pools take q as hi + lo halves, 22 bits.
//   p.v = (p s_v).(c - z) + sum_t p (b_v + z s_v), z = the middle code. These
// sums run over a whole segment, so their codes are centred by one packed
// subtraction: no offset to cancel, and terms of both signs.
// q is scaled by a power of two so that its largest element is in
// [2^13, 2^14): bf16 values then keep all their bits in fp16 down to 2^-27 of
// the largest. p s_v is scaled per group by a power of two kept across tiles
// (vinv) so that the largest |s_v| so far maps below 2^7 (with p up to
// 2^kSlack, p s_v stays below 2^15) and at 2^3 or above: scales of
// any magnitude neither overflow nor sink into fp16's subnormals. Split into hi
// + lo halves, a p s_v has 22 bits down to 2^-5 of the largest |s_v|, and below
// that an error of at most 2^-28 of it. One half alone was 13 bf16 ulp off where
// the terms of an output nearly cancel, and no faster.
// ---------------------------------------------------------------------------
template <typename E, int BITS, int D, int NB>
struct CodesAttend {
  using F = PagedFmt<sizeof(E), BITS, D>;
  static constexpr int NK = D / 16, NG = F::kGroups, NCH = F::kNChunk;
  static constexpr int KPC = NK / NCH;   // k-steps (and 16-dim output tiles) per 16-byte chunk: 1 or 2
  // Two blocks of heads take their tokens 16 at a time: with 32 they spill more at the register limit of 168 (heads of
  // 128 still do: bf16 176 bytes stored and 216 loaded), 4 x 128K in 8 bits 349 -> 303 us.
  static constexpr int MT = NB == 1 ? F::kTile / kPagedWarps / 16 : 1, PARTS = F::kTile / kPagedWarps / 16 / MT;
  static constexpr float MID = BITS == 8 ? 128.0f : 8.0f;
  static constexpr bool kOffset = __is_same(E, __nv_bfloat16), kOffsetLow = kOffset && BITS == 8;
  static constexpr int QT = sizeof(E) == 4 ? 2 : 1;  // fp16 terms of q
  uint32_t qb[QT][NB][NK][2];
  float qs[NB][2][NG], qoff[NB][2][NG], m[NB][2], l[NB][2], o[NB][NK][4], ob[NB][2][NG];
  float vinv[NG], vlim[NG], qfac;

  __device__ __forceinline__ void begin(const PagedParams& p, const float*, int b, int h, int, int lane) {
    const int g = lane >> 2, tq = lane & 3;
    // this lane's elements of head g: four (8-bit) or eight (4-bit) neighbours of every chunk
    constexpr int N = BITS == 8 ? 4 : 8, W = N * int(sizeof(E)) / 4;  // elements, 32-bit words
    uint32_t raw[NB][NCH][W];
    auto elements = [&](const uint32_t (&w)[W], float (&f)[N]) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (sizeof(E) == 4) f[i] = __uint_as_float(w[i]);
        else unpack_word<E>(w[i], f + 2 * i);
      }
    };
    float qmax = 0.0f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int hd = 8 * nb + g;
      const E* row = static_cast<const E*>(p.q) + (int64_t(b) * p.Hkv * p.G + int64_t(h) * p.G + hd) * D;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const uint32_t* at = reinterpret_cast<const uint32_t*>(row + F::kEpc * c + N * tq);
        if constexpr (W == 2) {
          const uint2 w = hd < p.G ? *reinterpret_cast<const uint2*>(at) : make_uint2(0, 0);
          raw[nb][c][0] = w.x, raw[nb][c][1] = w.y;
        } else {
#pragma unroll
          for (int i = 0; i < W; i += 4) {
            const uint4 w = hd < p.G ? *reinterpret_cast<const uint4*>(at + i) : make_uint4(0, 0, 0, 0);
            raw[nb][c][i] = w.x, raw[nb][c][i + 1] = w.y, raw[nb][c][i + 2] = w.z, raw[nb][c][i + 3] = w.w;
          }
        }
        float f[N];
        elements(raw[nb][c], f);
#pragma unroll
        for (int i = 0; i < N; ++i) qmax = fmaxf(qmax, fabsf(f[i]));
      }
    }
    qmax = warp_max(qmax);
    const int eq = qmax > 0.0f && qmax < INFINITY ? max(ilogbf(qmax) - 13, -126) : 0;
    const float up = exp2f(float(-eq));
    qfac = ldexpf(p.scale_log2, eq);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float sum[NG], off[NG];
#pragma unroll
      for (int r = 0; r < NG; ++r) sum[r] = off[r] = 0.0f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int r = c * F::kEpc / 64;
        float f[N];
        elements(raw[nb][c], f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sum[r] += f[i];
          f[i] *= up;
        }
        // k-slots {2tq, 2tq + 1} and {2tq + 8, 2tq + 9}, in the order in which the codes come out of a register
#pragma unroll
        for (int i = 0; i < KPC; ++i) {
          float x[2][2];
          if constexpr (BITS == 8) {
            x[0][0] = f[0], x[0][1] = f[1], x[1][0] = f[2], x[1][1] = f[3];
          } else {
            x[0][0] = f[2 * i], x[0][1] = f[2 * i + 4];
            x[1][0] = f[2 * i + 1] * 0.0625f, x[1][1] = f[2 * i + 5] * 0.0625f;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if constexpr (QT == 2) {
              split2<__half>(x[j][0], x[j][1], qb[0][nb][KPC * c + i][j], qb[QT - 1][nb][KPC * c + i][j]);
            } else {
              qb[0][nb][KPC * c + i][j] = pack2<__half>(x[j][0], x[j][1]);
              if (BITS == 8 || j == 1) {
                float g2[2];
                unpack_word<__half>(qb[0][nb][KPC * c + i][j], g2);
                off[r] += g2[0] + g2[1];
              }
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < NK; ++k) o[nb][k][0] = o[nb][k][1] = o[nb][k][2] = o[nb][k][3] = 0.0f;
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        off[r] += __shfl_xor_sync(0xffffffffu, off[r], 1);
        off[r] += __shfl_xor_sync(0xffffffffu, off[r], 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qs[nb][e][r] = p.scale_log2 * __shfl_sync(0xffffffffu, sum[r], 4 * (2 * tq + e));
          qoff[nb][e][r] = kOffset ? -1024.0f * __shfl_sync(0xffffffffu, off[r], 4 * (2 * tq + e)) : 0.0f;
          ob[nb][e][r] = 0.0f;
        }
      }
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.0f;
    }
#pragma unroll
    for (int r = 0; r < NG; ++r) {
      vinv[r] = 1.0f;
      vlim[r] = 0.0f;
    }
  }

  __device__ __forceinline__ void tile(const PagedParams& p, const float*, const TileView& t, int warp, int lane) {
#pragma unroll 1
    for (int i = 0; i < PARTS; ++i) part(p, t, (warp * PARTS + i) * 16 * MT, lane);
  }

  // Rows r0 .. r0 + 16 MT of the tile.
  __device__ __forceinline__ void part(const PagedParams& p, const TileView& t, int r0, int lane) {
    constexpr int TW = 16 * MT;
    const int g = lane >> 2, mq = lane >> 3, r8 = lane & 7;
    const int lo = t.lo - r0, hi = t.hi - r0;
    if (hi <= 0 || lo >= TW) return;
    const TileAddr<F> rows{smem_u32(t.stage), t.pb_log};
    const LaneAddr<F> la(8 * (mq & 1) + r8, mq >> 1);
    const bool whole = lo <= 0 && hi >= TW;
    const uint32_t magic = p.magic;
    const uint32_t ksc = smem_u32(t.stage) + 2 * F::kKvBytes + r0 * NG * int(sizeof(E));  // K scales; K biases, V scales, V biases follow
    const uint32_t kbi = ksc + F::kSbBytes, vsc = kbi + F::kSbBytes, vbi = vsc + F::kSbBytes;
    float s[MT][NB][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float acc[NG][NB][4];
#pragma unroll
      for (int r = 0; r < NG; ++r)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          acc[r][nb][0] = acc[r][nb][2] = qoff[nb][0][r];
          acc[r][nb][1] = acc[r][nb][3] = qoff[nb][1][r];
        }
#pragma unroll
      for (int c = 0; c < NCH; c += 2) {
        // matrices: tokens {0..7, 8..15} of chunks c and c + 1
        uint32_t a[4];
        ldsm_x4(la.at(rows.row_at(r0 + 16 * mt), c, t.pb_log), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < KPC; ++i) {
            const int k = (c + j) * KPC + i;
            const uint32_t x0 = a[2 * j], x1 = a[2 * j + 1];
            uint32_t f0, f1, f2, f3;
            if constexpr (BITS == 8) {
              f0 = raw_u8(x0, 0x5150u, magic), f1 = raw_u8(x1, 0x5150u, magic);
              f2 = raw_u8(x0, 0x5352u, magic), f3 = raw_u8(x1, 0x5352u, magic);
            } else {  // codes 2i, 2i + 4 (places 1) and 2i + 1, 2i + 5 (places 16) of the register
              f0 = raw_u4(x0 >> (8 * i), 0, magic), f1 = raw_u4(x1 >> (8 * i), 0, magic);
              f2 = raw_u4(x0 >> (8 * i), 1, magic), f3 = raw_u4(x1 >> (8 * i), 1, magic);
            }
            if constexpr (!kOffsetLow) f0 = sub_f16x2(f0, 0x64006400u), f1 = sub_f16x2(f1, 0x64006400u);
            if constexpr (!kOffset) f2 = sub_f16x2(f2, 0x64006400u), f3 = sub_f16x2(f3, 0x64006400u);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int t2 = 0; t2 < QT; ++t2)
                mma16816_f16(acc[k / 4][nb], f0, f1, f2, f3, qb[t2][nb][k][0], qb[t2][nb][k][1]);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int tk = 16 * mt + g + 8 * e;
        float ks[NG], kb[NG];
        load_groups<E, NG>(ksc, tk, ks);
        load_groups<E, NG>(kbi, tk, kb);
#pragma unroll
        for (int r = 0; r < NG; ++r) ks[r] *= qfac;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float v = 0.0f;
#pragma unroll
            for (int r = 0; r < NG; ++r)
              v = fmaf(ks[r], acc[r][nb][2 * e + hh], fmaf(kb[r], qs[nb][hh][r], v));
            s[mt][nb][2 * e + hh] = v;
          }
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tk = 16 * mt + g + 8 * (i >> 1);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[mt][nb][i] = tk < lo || tk >= hi ? -INFINITY : s[mt][nb][i];
        }
    }
    bool up = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) up |= s[mt][nb][i] > m[nb][i & 1] + kSlack;
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mx = fmaxf(mx, fmaxf(s[mt][nb][e], s[mt][nb][2 + e]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float f = raise_max(m[nb][e], mx);
          l[nb][e] *= f;
#pragma unroll
          for (int r = 0; r < NG; ++r) ob[nb][e][r] *= f;
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            o[nb][k][e] *= f;
            o[nb][k][2 + e] *= f;
          }
        }
      }
    }
    float vs[MT][2][NG], vb[MT][2][NG];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        load_groups<E, NG>(vsc, 16 * mt + g + 8 * e, vs[mt][e]);
        load_groups<E, NG>(vbi, 16 * mt + g + 8 * e, vb[mt][e]);
      }
    }
    if (!whole) {  // anything may lie past the end
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tk = 16 * mt + g + 8 * e;
#pragma unroll
          for (int r = 0; r < NG; ++r) {
            vs[mt][e][r] = tk < lo || tk >= hi ? 0.0f : vs[mt][e][r];
            vb[mt][e][r] = tk < lo || tk >= hi ? 0.0f : vb[mt][e][r];
          }
        }
    }
    float mu[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) mu[nb][hh] = m[nb][hh] == -INFINITY ? 0.0f : m[nb][hh];
    bool big = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int r = 0; r < NG; ++r) {
          vb[mt][e][r] = fmaf(MID, vs[mt][e][r], vb[mt][e][r]);
          big |= fabsf(vs[mt][e][r]) > vlim[r];
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const float pr = ex2(s[mt][nb][2 * e + hh] - mu[nb][hh]);
            s[mt][nb][2 * e + hh] = pr;
            l[nb][hh] += pr;
#pragma unroll
            for (int r = 0; r < NG; ++r) ob[nb][hh][r] = fmaf(pr, vb[mt][e][r], ob[nb][hh][r]);
          }
        }
      }
    }
    if (__any_sync(0xffffffffu, big)) {
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        float mx = 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) mx = fmaxf(mx, fmaxf(fabsf(vs[mt][0][r]), fabsf(vs[mt][1][r])));
        mx = warp_max(mx);
        if (mx > vlim[r] && mx < INFINITY) {
          const int e = max(ilogbf(mx), -100);
          const float inv = ldexpf(1.0f, 3 - e);
          const float f = vlim[r] > 0.0f ? inv / vinv[r] : 1.0f;  // o is still zero the first time
          vinv[r] = inv;
          vlim[r] = ldexpf(1.0f, min(e + 4, 127));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int k = 4 * r; k < 4 * r + 4; ++k)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[nb][k][i] *= f;
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t ph[NG][NB][2], pl[NG][NB][2];
#pragma unroll
      for (int r = 0; r < NG; ++r) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float sv = vs[mt][e][r] * vinv[r];
            uint32_t hi2, lo2;
            split2<__half>(s[mt][nb][2 * e] * sv, s[mt][nb][2 * e + 1] * sv, hi2, lo2);
            ph[r][nb][e] = movm_trans(hi2);
            pl[r][nb][e] = movm_trans(lo2);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < NCH; c += 2) {
        // matrices (transposed): tokens {0..7, 8..15} of chunks c and c + 1
        uint32_t a[4];
        ldsm_x4_t(la.at(rows.row_at(r0 + 16 * mt) + F::kKvBytes, c, t.pb_log), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < KPC; ++i) {
            const int k = (c + j) * KPC + i, r = k / 4;
            const uint32_t x0 = a[2 * j], x1 = a[2 * j + 1];
            uint32_t f0, f1, f2, f3;
            if constexpr (BITS == 8) {  // less 1024 + 128
              f0 = sub_f16x2(raw_u8(x0, 0x5250u, magic), 0x64806480u), f1 = sub_f16x2(raw_u8(x0, 0x5351u, magic), 0x64806480u);
              f2 = sub_f16x2(raw_u8(x1, 0x5250u, magic), 0x64806480u), f3 = sub_f16x2(raw_u8(x1, 0x5351u, magic), 0x64806480u);
            } else {  // less 1024 + 8, and 1024 + 16 * 8: rows g + 8 hold 16 (c - 8)
              f0 = sub_f16x2(raw_u4(x0 >> (8 * i), 0, magic), 0x64086408u), f1 = sub_f16x2(raw_u4(x0 >> (8 * i), 1, magic), 0x64806480u);
              f2 = sub_f16x2(raw_u4(x1 >> (8 * i), 0, magic), 0x64086408u), f3 = sub_f16x2(raw_u4(x1 >> (8 * i), 1, magic), 0x64806480u);
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              mma16816_f16(o[nb][k], f0, f1, f2, f3, ph[r][nb][0], ph[r][nb][1]);
              mma16816_f16(o[nb][k], f0, f1, f2, f3, pl[r][nb][0], pl[r][nb][1]);
            }
          }
        }
      }
    }
  }

  __device__ __forceinline__ void end(const PagedParams& p, const WarpPart<D>& w, int lane) {
    const int g = lane >> 2, tq = lane & 3;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float ls = l[nb][e];
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
          ls += __shfl_xor_sync(0xffffffffu, ls, x);
#pragma unroll
          for (int r = 0; r < NG; ++r) ob[nb][e][r] += __shfl_xor_sync(0xffffffffu, ob[nb][e][r], x);
        }
        const int hd = 8 * nb + 2 * tq + e;
        if (hd < p.G) {
          if (g == 0) {
            w.ml[2 * hd] = m[nb][e];
            w.ml[2 * hd + 1] = ls;
          }
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            const float back = 1.0f / vinv[k / 4];
            const int d = BITS == 8 ? 16 * k + 2 * g : 32 * (k >> 1) + 4 * g + 2 * (k & 1);
            *reinterpret_cast<float2*>(w.o + hd * (D + 4) + d) =
                make_float2(fmaf(o[nb][k][e], back, ob[nb][e][k / 4]),
                            fmaf(o[nb][k][2 + e], BITS == 8 ? back : back * 0.0625f, ob[nb][e][k / 4]));
          }
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------
// Dense fp32 pools on the FMA pipes: the tensor cores have no fp32 product. A
// warp has 8 tokens of a tile and HB blocks of four heads. q.k: lane = (token,
// head), so a score needs no exchange and no array over heads, which keeps the
// code short -- a small call spends more on fetching instructions than on
// executing them. p.v: lane = (head, every eighth chunk of the row), p from the
// score's lane by one shuffle per token. Keys and values are read once for all
// heads. q (times scale * log2 e, rows padded against bank conflicts) lies in
// shared memory.
// ---------------------------------------------------------------------------
template <int D, int HB>
struct FmaAttend {
  using F = PagedFmt<4, 0, D>;
  static constexpr int NCH = F::kNChunk, TW = 8, DL = D / 8;
  static_assert(F::kTile == TW * kPagedWarps && F::kBoxBytes == 128, "eight tokens per warp, whole swizzle rows");
  float m[HB], l[HB], o[HB][DL];  // of head 4 hb + lane % 4 (m, l) and 4 hb + lane / 8 (o)

  // Where a lane's dims lie in the row: every eighth chunk, so that the eight lanes of a head read all banks.
  static __device__ __forceinline__ int dim(int lane, int i) { return 4 * (8 * (i / 4) + (lane & 7)) + i % 4; }

  // every consumer thread calls; qf: [G][D + 4]
  __device__ __forceinline__ void begin(const PagedParams& p, float* qf, int b, int h, int warp, int lane) {
    const float* q = static_cast<const float*>(p.q) + (int64_t(b) * p.Hkv * p.G + int64_t(h) * p.G) * D;
#pragma unroll 1
    for (int i = warp * 32 + lane; i < p.G * D; i += 32 * kPagedWarps)
      qf[i / D * (D + 4) + i % D] = q[i] * p.scale_log2;
    named_barrier(1, 32 * kPagedWarps);
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
      m[hb] = -INFINITY;
      l[hb] = 0.0f;
#pragma unroll
      for (int i = 0; i < DL; ++i) o[hb][i] = 0.0f;
    }
  }

  __device__ __forceinline__ void tile(const PagedParams& p, const float* qf, const TileView& t, int warp, int lane) {
    const int r0 = warp * TW;
    const int lo = max(t.lo - r0, 0), hi = min(t.hi - r0, TW);
    if (hi <= lo) return;
    const int tok = lane >> 2, vh = lane >> 3;  // q.k: (tok, lane % 4); p.v: (vh, dims)
    const bool ok = tok >= lo && tok < hi;
    // chunk c of row r of the eight lies at rows + (c / 8) box + 128 r + 16 ((c % 8) ^ r)
    const uint32_t rows = TileAddr<F>{smem_u32(t.stage), t.pb_log}.row_at(r0), box = 128u << t.pb_log;
    const uint32_t krow = rows + tok * 128, vrows = rows + F::kKvBytes;
    const float* qrow[HB];
    float s[HB];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
      qrow[hb] = qf + min(4 * hb + (lane & 3), p.G - 1) * (D + 4);  // a head past the last repeats it
      s[hb] = 0.0f;
    }
#pragma unroll 4
    for (int c = 0; c < NCH; ++c) {
      const float4 x = lds_f4(krow + (c / 8) * box + (((c % 8) ^ tok) << 4));
#pragma unroll
      for (int hb = 0; hb < HB; ++hb) {
        const float4 y = *reinterpret_cast<const float4*>(qrow[hb] + 4 * c);
        s[hb] += fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, x.x * y.x)));
      }
    }
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
      s[hb] = ok ? s[hb] : -INFINITY;
      if (__any_sync(0xffffffffu, s[hb] > m[hb] + kSlack)) {
        float mx = s[hb];
        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        float f = raise_max(m[hb], mx);
        l[hb] *= f;
        f = __shfl_sync(0xffffffffu, f, vh);  // lane vh holds head vh's
#pragma unroll
        for (int i = 0; i < DL; ++i) o[hb][i] *= f;
      }
      s[hb] = exp2_from(s[hb], m[hb]);
      l[hb] += s[hb];
    }
#pragma unroll 2
    for (int tk = lo; tk < hi; ++tk) {
      float v[DL];
      const uint32_t at = vrows + tk * 128 + (((lane & 7) ^ tk) << 4);
#pragma unroll
      for (int c = 0; c < DL / 4; ++c) {
        const float4 x = lds_f4(at + c * box);
        v[4 * c] = x.x, v[4 * c + 1] = x.y, v[4 * c + 2] = x.z, v[4 * c + 3] = x.w;
      }
#pragma unroll
      for (int hb = 0; hb < HB; ++hb) {
        const float pr = __shfl_sync(0xffffffffu, s[hb], 4 * tk + vh);
#pragma unroll
        for (int i = 0; i < DL; ++i) o[hb][i] = fmaf(pr, v[i], o[hb][i]);
      }
    }
  }

  __device__ __forceinline__ void end(const PagedParams& p, const WarpPart<D>& w, int lane) {
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
      float ls = l[hb];
      for (int x = 4; x < 32; x <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, x);
      const int hd = 4 * hb + (lane & 3), vh = 4 * hb + (lane >> 3);
      if (lane < 4 && hd < p.G) {
        w.ml[2 * hd] = m[hb];
        w.ml[2 * hd + 1] = ls;
      }
      if (vh < p.G) {
#pragma unroll
        for (int i = 0; i < DL; i += 4)
          *reinterpret_cast<float4*>(w.o + vh * (D + 4) + dim(lane, i)) =
              make_float4(o[hb][i], o[hb][i + 1], o[hb][i + 2], o[hb][i + 3]);
      }
    }
  }
};

// ---------------------------------------------------------------------------
// The line of tiles and a CTA's walk over its piece
// ---------------------------------------------------------------------------

// Tokens [begin, end) that sequence b attends to.
struct TokenRange { int begin, end; };
__device__ __forceinline__ TokenRange token_range(const PagedParams& p, int b) {
  const int64_t cap = int64_t(p.W) * p.P;
  const int raw = __ldcg(p.lengths + b);  // from L2: the merge reads it before its wait
  if ((raw < 0 || raw > cap) && p.flags && blockIdx.x == 0) atomicOr(p.flags, kErrBadIndex);
  const int len = raw < 0 ? 0 : raw > cap ? int(cap) : raw;
  return {p.window > 0 && len > p.window ? len - p.window : 0, len};
}
// Units of one pair on the line: kSegmentUnits for beginning and ending its
// segment, then one per tile; none if it has no tokens.
__device__ __forceinline__ int units_of(TokenRange r, int tile) {
  return r.end > r.begin ? (r.end + tile - 1) / tile - r.begin / tile + kSegmentUnits : 0;
}

// The line of U units in equal pieces for the CTAs that take part: the first
// `rem` pieces have base + 1 units. Small calls give every CTA two units
// rather than one: half as many segments to join (one bf16 sequence of 2K
// tokens 8.4 -> 7.6 us; with three or four 7.9, 8.3).
struct Pieces {
  int n, base, rem;
  __device__ __forceinline__ Pieces(const PagedParams& p, int U) {
    n = min((U + 1) / 2, p.ncta);
    base = n ? U / n : 0;
    rem = U - base * n;
  }
  __device__ __forceinline__ int begin(int c) const { return c * base + min(c, rem); }
  __device__ __forceinline__ int of(int u) const {  // the piece that holds unit u
    const int big = rem * (base + 1);
    return u < big ? u / (base + 1) : rem + (u - big) / base;
  }
};

struct Segment {
  int b, h;
  int i0, i1, nt;  // tiles [i0, i1) of the pair's nt
};

struct Walk {
  const int* prefix;
  int Hkv, b, u, u1;
  __device__ __forceinline__ Walk(const int* pre, int B, int hkv, int begin, int end)
      : prefix(pre), Hkv(hkv), b(0), u(begin), u1(end) {
    int lo = 0, hi = B;  // the largest b with prefix[b] * Hkv <= u; a b without tiles is passed over
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] * Hkv <= u) lo = mid; else hi = mid;
    }
    b = lo;
  }
  __device__ __forceinline__ bool next(Segment& s) {
    while (u < u1) {
      while (prefix[b + 1] * Hkv <= u) ++b;  // ends: u < prefix[B] * Hkv
      const int nu = prefix[b + 1] - prefix[b], r = u - prefix[b] * Hkv;
      s.b = b;
      s.h = r / nu;
      s.nt = nu - kSegmentUnits;
      const int first = r - s.h * nu, last = min(nu, first + u1 - u);
      u += last - first;
      s.i0 = max(first - kSegmentUnits, 0);
      s.i1 = last - kSegmentUnits;
      if (s.i1 > s.i0) return true;
    }
    return false;
  }
};

// NB: blocks of heads, of four for dense fp32 pools, else of eight.
template <typename E, int BITS, int D, int NB>
struct PickAttend { using type = CodesAttend<E, BITS, D, NB>; };
template <typename E, int D, int NB>
struct PickAttend<E, 0, D, NB> { using type = DenseAttend<E, D, NB>; };
template <int D, int NB>
struct PickAttend<float, 0, D, NB> { using type = FmaAttend<D, NB>; };

// After a wait that expired: wait, with the limit, for the copies of the last
// `stages` of `it` uses, which still land in this CTA's shared memory.
static __device__ __noinline__ void drain(uint64_t* full, int it, int stages) {
  for (int k = max(0, it - stages); k < it; ++k) mbar_wait(full + k % stages, uint32_t(k / stages) & 1u, nullptr);
}

// The producer warp: this CTA's tiles into the ring, stage by stage.
template <typename E, int BITS, int D>
__device__ __forceinline__ void paged_produce(const PagedParams& p, const CUtensorMap* tmK, const CUtensorMap* tmV,
                                              uint8_t* ring, uint64_t* full, uint64_t* empty, Walk walk, int lane) {
  using F = PagedFmt<sizeof(E), BITS, D>;
  const uint64_t pol = stream_policy(false);
  const int pb = min(p.P, F::kTile), nb = F::kTile / pb;   // rows per box, boxes per tile
  const int p_log = __ffs(p.P) - 1, pb_log = __ffs(pb) - 1;
  const int oob_row = int(p.n_pages * p.Hkv * p.P);  // past the tensor: TMA fills zeros
  int it = 0, st = 0;
  uint32_t round = 0;  // parity of the stages' current use
  Segment s;
  while (walk.next(s)) {
    const TokenRange r = token_range(p, s.b);
    const int* row = p.tables + int64_t(s.b) * p.W;
    const int t0 = r.begin / F::kTile;
    const int last_slot = (r.end - 1) >> p_log, first_slot = r.begin >> p_log;
    auto load = [&](int slot) { return slot >= first_slot && slot <= last_slot ? row[slot] : -1; };
    int base = ((t0 + s.i0) * F::kTile) >> p_log;
    int cur = load(base + lane), nxt = load(base + 32 + lane);
    for (int i = s.i0; i < s.i1; ++i, ++it) {
      const int tok = (t0 + i) * F::kTile;
      if ((tok >> p_log) - base >= 32) {
        base += 32;
        cur = nxt;
        nxt = load(base + 32 + lane);
      }
      // lane j < nb: the page of box j (-1: no token of the range lies in it)
      const int tj = tok + (lane < nb ? lane : 0) * pb;
      const int off = (tj >> p_log) - base;
      const int a = __shfl_sync(0xffffffffu, cur, off & 31), c = __shfl_sync(0xffffffffu, nxt, off & 31);
      int page = off < 32 ? a : c;
      const bool need = lane < nb && tj < r.end && tj + pb > r.begin;
      bool bad = false;
      if (need && (page < 0 || page >= p.n_pages)) {
        bad = true;
        if (p.flags) atomicOr(p.flags, kErrBadIndex);
      }
      const int n_box = __popc(__ballot_sync(0xffffffffu, need));
      const int64_t krow = (int64_t(page) * p.Hkv + s.h) * p.P + (tj & (p.P - 1));
      if (it >= p.stages && !mbar_wait(empty + st, round ^ 1u, p.flags)) {
        // the consumers gave up: no more copies, but those under way must land before this CTA may end
        drain(full, it, p.stages);
        return;
      }
      uint8_t* stage = ring + st * F::kStageBytes;
      if (lane == 0) mbar_arrive_expect_tx(full + st, uint32_t(n_box * 2 * pb * F::kRowBytes));
      __syncwarp();
      if (need) {
        const int y = bad ? oob_row : int(krow);
        uint8_t* dst = stage + lane * pb * F::kRowBytes;
        tma_load_3d(dst, tmK, 0, y, 0, full + st, pol);
        tma_load_3d(dst + F::kKvBytes, tmV, 0, y, 0, full + st, pol);
      }
      if constexpr (BITS != 0) {
        constexpr int ROW = F::kGroups * int(sizeof(E));     // bytes of a token in each scale/bias array
        constexpr int CPA = F::kSbBytes / 16;                // chunks of a stage in each array
        const uint8_t* src[4] = {static_cast<const uint8_t*>(p.k_scales), static_cast<const uint8_t*>(p.k_biases),
                                 static_cast<const uint8_t*>(p.v_scales), static_cast<const uint8_t*>(p.v_biases)};
        const int good = need && !bad ? 1 : 0;
        const uint32_t sb = smem_u32(stage + 2 * F::kKvBytes);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
          for (int k = 0; k < CPA; k += 32) {
            const int c2 = k + lane, byte = c2 * 16;
            const int j = min((byte / ROW) >> pb_log, nb - 1);  // the box this chunk's tokens lie in
            const int64_t kr = __shfl_sync(0xffffffffu, krow, j);
            const int g2 = __shfl_sync(0xffffffffu, good, j);
            if (c2 < CPA)
              cp_async16_zfill(sb + x * F::kSbBytes + byte, g2 ? src[x] + (kr * ROW + byte - j * pb * ROW) : src[x],
                               g2 ? 16 : 0);
          }
        }
        cp_async_arrive(full + st);
      }
      if (++st == p.stages) {
        st = 0;
        round ^= 1u;
      }
    }
  }
}

template <typename E, int BITS, int D, int NB>
__global__ void __launch_bounds__(kPagedThreads, 2)
paged_decode_kernel(const __grid_constant__ PagedParams p, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV) {
  using F = PagedFmt<sizeof(E), BITS, D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* qf = reinterpret_cast<float*>(sm + p.q_off);
  float* buf = reinterpret_cast<float*>(sm + p.buf_off);
  int* prefix = reinterpret_cast<int*>(sm + p.prefix_off);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + p.bar_off);
  uint64_t* empty = full + kPagedMaxStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full + i, BITS ? 33 : 1);
      mbar_init(empty + i, kPagedWarps);
    }
    fence_mbar_init();
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  // The merge may start from here on: what ran before this kernel is complete then, so that it may read the lengths.
  griddep_wait();
  griddep_launch_dependents();

  // units of the line before each sequence (of one kv head)
  if (p.B < 32) {  // every warp for itself: no barrier on the way to the first copy
    prefix += warp * 32;
    int incl = lane < p.B ? units_of(token_range(p, lane), F::kTile) : 0;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, x);
      if (lane >= x) incl += v;
    }
    const int before = __shfl_up_sync(0xffffffffu, incl, 1);
    prefix[lane] = lane ? before : 0;  // B + 1 entries matter
    __syncthreads();                   // the barriers of the ring are set up, too
  } else {
    int* warp_tot = prefix + p.B + 1;
    const int per = (p.B + kPagedThreads - 1) / kPagedThreads;
    int mine = 0;
    for (int k = 0; k < per; ++k) {
      const int b = tid * per + k;
      if (b < p.B) mine += units_of(token_range(p, b), F::kTile);
    }
    int incl = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, x);
      if (lane >= x) incl += v;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    int run = incl - mine;
    for (int w = 0; w < warp; ++w) run += warp_tot[w];
    for (int k = 0; k < per; ++k) {
      const int b = tid * per + k;
      if (b < p.B) {
        prefix[b] = run;
        run += units_of(token_range(p, b), F::kTile);
        if (b == p.B - 1) prefix[p.B] = run;
      }
    }
    __syncthreads();
  }

  const Pieces pieces(p, prefix[p.B] * p.Hkv);
  if (int(blockIdx.x) >= pieces.n) return;
  Walk walk(prefix, p.B, p.Hkv, pieces.begin(blockIdx.x), pieces.begin(blockIdx.x + 1));

  if (warp == kPagedWarps) {
    paged_produce<E, BITS, D>(p, &tmK, &tmV, sm, full, empty, walk, lane);
    return;
  }
  using A = typename PickAttend<E, BITS, D, NB>::type;
  const int pb_log = __ffs(min(p.P, F::kTile)) - 1;
  A att;
  Segment s;
  int it = 0, st = 0;
  uint32_t round = 0;
  bool dead = false, first = true;
  while (walk.next(s)) {
    const TokenRange r = token_range(p, s.b);
    const int t0 = r.begin / F::kTile;
    att.begin(p, qf, s.b, s.h, warp, lane);
    for (int i = s.i0; i < s.i1; ++i, ++it) {
      const int tok = (t0 + i) * F::kTile;
      if (!dead) dead = !mbar_wait(full + st, round, p.flags);
      if (!dead) {
        att.tile(p, qf, TileView{sm + st * F::kStageBytes, pb_log, r.begin - tok, r.end - tok}, warp, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + st);
      }
      if (++st == p.stages) {
        st = 0;
        round ^= 1u;
      }
    }
    att.end(p, WarpPart<D>(buf, p.G, warp), lane);
    named_barrier(1, 32 * kPagedWarps);
    // the four warps' parts, in warp order
    const bool whole = s.i0 == 0 && s.i1 == s.nt;
    float* part = p.part + (int64_t(blockIdx.x) * 2 + (first ? 0 : 1)) * paged_part_floats(p.G, D);
    for (int k = tid; k < p.G * (D / 4); k += 32 * kPagedWarps) {
      const int g = k / (D / 4), d = (k % (D / 4)) * 4;
      float mw[kPagedWarps], M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        mw[w] = WarpPart<D>(buf, p.G, w).ml[2 * g];
        M = fmaxf(M, mw[w]);
      }
      float4 O = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        const WarpPart<D> wp(buf, p.G, w);
        const float f = exp2_from(mw[w], M);
        const float4 x = *reinterpret_cast<const float4*>(wp.o + g * (D + 4) + d);
        L = fmaf(f, wp.ml[2 * g + 1], L);
        O.x = fmaf(f, x.x, O.x);
        O.y = fmaf(f, x.y, O.y);
        O.z = fmaf(f, x.z, O.z);
        O.w = fmaf(f, x.w, O.w);
      }
      if (whole) {
        const int hq = s.h * p.G + g;
        if (p.sinks) L += exp2f(fmaf(p.sinks[hq], 1.4426950408889634f, -(M == -INFINITY ? 0.0f : M)));
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        E* out = static_cast<E*>(p.out) + (int64_t(s.b) * p.Hkv * p.G + hq) * D + d;
        if constexpr (sizeof(E) == 4) {
          *reinterpret_cast<float4*>(out) = make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
        } else {
          *reinterpret_cast<uint2*>(out) = make_uint2(pack2<E>(O.x * inv, O.y * inv), pack2<E>(O.z * inv, O.w * inv));
        }
      } else {
        *reinterpret_cast<float4*>(part + g * D + d) = O;
        if (d == 0) {
          part[p.G * D + 2 * g] = M;
          part[p.G * D + 2 * g + 1] = L;
        }
      }
    }
    named_barrier(1, 32 * kPagedWarps);
    first = false;
  }
  if (dead) drain(full, it, p.stages);
}

// Joins the segments of HB query heads of one sequence (grid: B * ceil(Hq / HB)
// blocks) in a fixed order; a pair that one CTA did alone is already written,
// an empty one is written here as zeros. Bound by the latency of its dependent
// loads, not by their bytes (a few MB at most, from L2): a lane takes the
// (m, l) of one segment each, and the o rows are loaded eight at a time, the
// first eight before the weights are known. Warps share a head's segments
// (warp w: w, w + 8, ...), except that with HB = 8 they take a head each where
// no pair has more than 32 segments.
template <typename E, int D, int TILE, int HB>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const __grid_constant__ PagedParams p) {
  constexpr int NW = kMergeThreads / 32, V = D / 32, BATCH = 8;
  static_assert(HB == 1 || HB == NW, "a warp per head, or all for one");
  __shared__ float red[NW][D], top[NW], tot[NW];
  __shared__ int sums[NW][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Hq = p.Hkv * p.G, per = (Hq + HB - 1) / HB, b = blockIdx.x / per;
  const int h0 = (blockIdx.x - b * per) * HB, h1 = min(h0 + HB, Hq);  // query heads
  // The sequence's place on the line, from the lengths, while the segments are still being worked on.
  int pre = 0, all = 0;
  for (int i = tid; i < p.B; i += kMergeThreads) {
    const int n = units_of(token_range(p, i), TILE);
    all += n;
    pre += i < b ? n : 0;
  }
  pre = __reduce_add_sync(0xffffffffu, pre);
  all = __reduce_add_sync(0xffffffffu, all);
  if (lane == 0) sums[warp][0] = pre, sums[warp][1] = all;
  __syncthreads();
  pre = all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) pre += sums[w][0], all += sums[w][1];
  const int nu = units_of(token_range(p, b), TILE);
  const Pieces pieces(p, all * p.Hkv);
  struct Place { int g, c0, ns, skip; };  // head of its pair; the pair's first CTA, its segments, the slot of the first
  auto place = [&](int hq) {
    const int h = hq / p.G, a = pre * p.Hkv + h * nu;  // the pair's first unit
    const int c0 = pieces.of(a + kSegmentUnits), c1 = pieces.of(a + nu - 1);  // with tiles of it
    // a CTA leaves its first segment in slot 0: the pair is that for all but, perhaps, c0
    return Place{hq - h * p.G, c0, c1 - c0 + 1, pieces.begin(c0) < a ? 1 : 0};
  };
  const int mine = HB > 1 ? min(h0 + warp, h1 - 1) : h0;
  Place at = {};
  if (nu != 0) at = place(mine);
  griddep_wait();
  E* out = static_cast<E*>(p.out) + int64_t(b) * Hq * D;
  if (nu == 0) {
    for (int d = h0 * D + tid; d < h1 * D; d += kMergeThreads) out[d] = Elt<E>::from_f32(0.0f);
    return;
  }
  const int stride = paged_part_floats(p.G, D);

  // Segments first, first + step, ... of the head at `at` joined into M, L, acc
  // (o of elements lane * V ...); false: its pair has one segment.
  auto join = [&](const Place& at, int first, int step, float& M, float& L, float (&acc)[V]) {
    const int g = at.g, ns = at.ns;
    if (ns == 1) return false;
    auto slot = [&](int i) { return p.part + (int64_t(at.c0 + i) * 2 + (i == 0 ? at.skip : 0)) * stride; };
    M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    for (int base = first; base < ns; base += 32 * step) {  // lane j: segment base + j * step
      const int n = min(32, (ns - base + step - 1) / step);
      float2 ml = make_float2(-INFINITY, 0.0f);
      if (lane < n) ml = *reinterpret_cast<const float2*>(slot(base + lane * step) + p.G * D + 2 * g);
      float x[BATCH][V];
      auto load = [&](int j0) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          if (j0 + j < n) {
            const float* o = slot(base + (j0 + j) * step) + g * D + lane * V;
            if constexpr (V == 4) {
              const float4 y = *reinterpret_cast<const float4*>(o);
              x[j][0] = y.x, x[j][1] = y.y, x[j][2] = y.z, x[j][3] = y.w;
            } else {
              const float2 y = *reinterpret_cast<const float2*>(o);
              x[j][0] = y.x, x[j][1] = y.y;
            }
          }
        }
      };
      load(0);
      const float f0 = raise_max(M, warp_max(ml.x)), f = exp2_from(ml.x, M);
      L = fmaf(L, f0, warp_sum(f * ml.y));
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= f0;
      for (int j0 = 0; j0 < n; j0 += BATCH) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const float w = __shfl_sync(0xffffffffu, f, (j0 + j) & 31);
          if (j0 + j < n) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = fmaf(w, x[j][i], acc[i]);
          }
        }
        load(j0 + BATCH);
      }
    }
    return true;
  };
  auto sink = [&](int hq, float M) {
    return p.sinks ? exp2f(fmaf(p.sinks[hq], 1.4426950408889634f, -(M == -INFINITY ? 0.0f : M))) : 0.0f;
  };

  float M, L, acc[V];
  if (HB > 1 && nu / pieces.base + 2 <= 32) {  // at least the segments of a pair of nu units
    const int hq = h0 + warp;
    if (hq >= h1 || !join(at, 0, 1, M, L, acc)) return;
    L += sink(hq, M);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] *= inv;
    E* row = out + hq * D + lane * V;
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < V; i += 2) *reinterpret_cast<float2*>(row + i) = make_float2(acc[i], acc[i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(row + i) = pack2<E>(acc[i], acc[i + 1]);
    }
    return;
  }
#pragma unroll 1
  for (int hq = h0; hq < h1; ++hq) {
    if (HB > 1) at = place(hq);
    if (!join(at, warp, NW, M, L, acc)) continue;  // alike for all threads
#pragma unroll
    for (int i = 0; i < V; ++i) red[warp][lane * V + i] = acc[i];
    if (lane == 0) {
      top[warp] = M;
      tot[warp] = L;
    }
    __syncthreads();
    if (tid < D) {  // D <= kMergeThreads
      M = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, top[w]);
      float O = 0.0f;
      L = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = exp2_from(top[w], M);
        L = fmaf(f, tot[w], L);
        O = fmaf(f, red[w][tid], O);
      }
      L += sink(hq, M);
      out[hq * D + tid] = Elt<E>::from_f32(L == 0.0f ? 0.0f : O / L);
    }
    if (HB > 1) __syncthreads();
  }
}

}  // namespace sd
