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
// depend on timing. The lengths are read on the device only, so a captured
// graph serves growing sequences.
//
// The running maximum m is a lower bound of the true one by at most kSlack
// (log2 units): it moves, and l and o are rescaled, only when a score passes
// m + kSlack, which one vote per tile finds; p stays below 2^kSlack.
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
  __device__ __forceinline__ uint32_t at(int row, int chunk) const {
    const int pb = 1 << pb_log;
    return base + uint32_t((row >> pb_log) * (pb * F::kRowBytes) + (chunk / F::kCpb) * (pb * F::kBoxBytes)) +
           swz(uint32_t((row & (pb - 1)) * F::kBoxBytes + (chunk % F::kCpb) * 16), F::kCpb);
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

__device__ __forceinline__ float exp2_from(float s, float m) { return exp2f(s - (m == -INFINITY ? 0.0f : m)); }

// New running maximum and the factor for what was summed under the old one.
__device__ __forceinline__ float raise_max(float& m, float mx) {
  const float mn = fmaxf(m, mx);
  const float f = mn == -INFINITY ? 1.0f : exp2f(m - mn);
  m = mn;
  return f;
}

// ---------------------------------------------------------------------------
// 16-bit K and V on the tensor cores, tokens as the rows of the tile:
// S^T = K q^T (m16n8k16: 16 tokens x 8 heads), O^T = V^T P^T (16 dims x 8
// heads). G <= 8 heads fill the 8 columns of one block, up to 16 two blocks.
// Lane (g, tq) = (lane / 4, lane % 4): S^T rows g, g + 8 are tokens and its
// columns 2tq, 2tq + 1 heads, the same heads as in O^T, so the softmax state
// of a head lies where its outputs are. P^T gets its operand layout from
// movmatrix. p is used as hi + lo halves of the element type (about 16 bits
// of it for bf16): a single bf16 p would cost as much accuracy as the final
// rounding does, and the extra mma is free next to the loads.
// ---------------------------------------------------------------------------
template <typename E, int D, int NB>
struct DenseAttend {
  using F = PagedFmt<2, 0, D>;
  static constexpr int NC = D / 16;
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
        qb[nb][c][0] = hd < p.G ? __ldg(q + row + 8 * c + tq) : 0u;
        qb[nb][c][1] = hd < p.G ? __ldg(q + row + 8 * c + 4 + tq) : 0u;
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
    const TileAddr<F> ka{smem_u32(t.stage), t.pb_log}, va{smem_u32(t.stage) + F::kKvBytes, t.pb_log};
    float acc[2][NB][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) acc[i][nb][0] = acc[i][nb][1] = acc[i][nb][2] = acc[i][nb][3] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t a0, a1, a2, a3;
      ldsm_x4(ka.at(r0 + 8 * (mq & 1) + r8, 2 * c + (mq >> 1)), a0, a1, a2, a3);
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
        up |= s[nb][i] > m[nb][i & 1] + kSlack;
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
          const float f = raise_max(m[nb][e], mx);
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
      ldsm_x4_t(va.at(r0 + 8 * (mq >> 1) + r8, 2 * c + (mq & 1)), a0, a1, a2, a3);
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

// Scales (or biases) of token t for every group, in fp32; zeros if !ok.
template <typename E, int NG>
__device__ __forceinline__ void load_groups(const E* a, int t, bool ok, float (&f)[NG]) {
  if constexpr (NG == 2) {
    unpack_word<E>(ok ? reinterpret_cast<const uint32_t*>(a)[t] : 0u, f);
  } else {
    f[0] = ok ? Elt<E>::to_f32(a[t]) : 0.0f;
  }
}

// ---------------------------------------------------------------------------
// 4/8-bit codes with 16-bit scales, the same products. The codes enter as
// exact fp16 integers (code_pair_u8 / code_pair_u4):
//   q.k = s_k (q.c) + b_k sum(q)             per 64-dim group, in fp32
//   p.v = (p s_v).c + sum_t p b_v
// q is scaled by a power of two so that its largest element is in
// [2^13, 2^14): bf16 values then keep all their bits in fp16 down to 2^-27 of
// the largest. p s_v is scaled per group by a power of two kept across tiles
// (vinv) so that the largest |s_v| so far maps near 2^6: hi + lo fp16 halves
// hold it to about 22 bits, and values of any magnitude neither overflow nor
// sink into fp16's subnormals.
// ---------------------------------------------------------------------------
template <typename E, int BITS, int D, int NB>
struct CodesAttend {
  using F = PagedFmt<2, BITS, D>;
  static constexpr int NK = D / 16, NG = F::kGroups, NCH = F::kNChunk;
  static constexpr int KPC = NK / NCH;   // k-steps (and 16-dim output tiles) per 16-byte chunk: 1 or 2
  static constexpr int MT = F::kTile / kPagedWarps / 16;
  uint32_t qb[NB][NK][2];
  float qs[NB][2][NG], m[NB][2], l[NB][2], o[NB][NK][4], ob[NB][2][NG];
  float vinv[NG], vlim[NG], qfac;

  // dims of k-slot pairs {2tq, 2tq + 1} and {2tq + 8, 2tq + 9} of k-step k
  static __device__ __forceinline__ void dims(int k, int tq, int (&d)[4]) {
    if constexpr (BITS == 8) {
      const int d0 = 16 * k + 4 * tq;
      d[0] = d0, d[1] = d0 + 1, d[2] = d0 + 2, d[3] = d0 + 3;
    } else {
      const int d0 = 32 * (k >> 1) + 8 * tq + 2 * (k & 1);
      d[0] = d0, d[1] = d0 + 4, d[2] = d0 + 1, d[3] = d0 + 5;
    }
  }

  __device__ __forceinline__ void begin(const PagedParams& p, const float*, int b, int h, int, int lane) {
    const int g = lane >> 2, tq = lane & 3;
    const E* q = static_cast<const E*>(p.q);
    float qmax = 0.0f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int hd = 8 * nb + g;
      const E* row = q + (int64_t(b) * p.Hkv * p.G + int64_t(h) * p.G + hd) * D;
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        int d[4];
        dims(k, tq, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) qmax = fmaxf(qmax, hd < p.G ? fabsf(Elt<E>::to_f32(__ldg(row + d[i]))) : 0.0f);
      }
    }
    qmax = warp_max(qmax);
    const int eq = qmax > 0.0f && qmax < INFINITY ? ilogbf(qmax) - 13 : 0;
    const float up = exp2f(float(-eq));
    qfac = ldexpf(p.scale_log2, eq);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int hd = 8 * nb + g;
      const E* row = q + (int64_t(b) * p.Hkv * p.G + int64_t(h) * p.G + hd) * D;
      float sum[NG];
#pragma unroll
      for (int r = 0; r < NG; ++r) sum[r] = 0.0f;
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        int d[4];
        dims(k, tq, d);
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[i] = hd < p.G ? Elt<E>::to_f32(__ldg(row + d[i])) : 0.0f;
          sum[k / 4] += f[i];
          f[i] *= up;
        }
        qb[nb][k][0] = pack2<__half>(f[0], f[1]);
        qb[nb][k][1] = pack2<__half>(f[2], f[3]);
        o[nb][k][0] = o[nb][k][1] = o[nb][k][2] = o[nb][k][3] = 0.0f;
      }
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qs[nb][e][r] = p.scale_log2 * __shfl_sync(0xffffffffu, sum[r], 4 * (2 * tq + e));
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

  __device__ __forceinline__ void tile(const PagedParams&, const float*, const TileView& t, int warp, int lane) {
    constexpr int TW = 16 * MT;
    const int g = lane >> 2, mq = lane >> 3, r8 = lane & 7;
    const int r0 = warp * TW;
    const int lo = t.lo - r0, hi = t.hi - r0;
    if (hi <= 0 || lo >= TW) return;
    const TileAddr<F> ka{smem_u32(t.stage), t.pb_log}, va{smem_u32(t.stage) + F::kKvBytes, t.pb_log};
    const E* ksc = reinterpret_cast<const E*>(t.stage + 2 * F::kKvBytes) + r0 * NG;
    const E *kbi = ksc + F::kTile * NG, *vsc = ksc + 2 * F::kTile * NG, *vbi = ksc + 3 * F::kTile * NG;
    float s[MT][NB][4];
    bool up = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float acc[NG][NB][4];
#pragma unroll
      for (int r = 0; r < NG; ++r)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[r][nb][0] = acc[r][nb][1] = acc[r][nb][2] = acc[r][nb][3] = 0.0f;
#pragma unroll
      for (int c = 0; c < NCH; c += 2) {
        // matrices: tokens {0..7, 8..15} of chunks c and c + 1
        uint32_t a[4];
        ldsm_x4(ka.at(r0 + 16 * mt + 8 * (mq & 1) + r8, c + (mq >> 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < KPC; ++i) {
            const int k = (c + j) * KPC + i;
            const uint32_t x0 = a[2 * j], x1 = a[2 * j + 1];
            uint32_t f0, f1, f2, f3;
            if constexpr (BITS == 8) {
              f0 = code_pair_u8(x0, 0x4140u), f1 = code_pair_u8(x1, 0x4140u);
              f2 = code_pair_u8(x0, 0x4342u), f3 = code_pair_u8(x1, 0x4342u);
            } else {
              f0 = code_pair_u4(x0, 2 * i), f1 = code_pair_u4(x1, 2 * i);
              f2 = code_pair_u4(x0, 2 * i + 1), f3 = code_pair_u4(x1, 2 * i + 1);
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              mma16816_f16(acc[k / 4][nb], f0, f1, f2, f3, qb[nb][k][0], qb[nb][k][1]);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int tk = 16 * mt + g + 8 * e;
        const bool ok = tk >= lo && tk < hi;
        float ks[NG], kb[NG];
        load_groups<E, NG>(ksc, tk, ok, ks);
        load_groups<E, NG>(kbi, tk, ok, kb);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float v = 0.0f;
#pragma unroll
            for (int r = 0; r < NG; ++r)
              v = fmaf(ks[r], acc[r][nb][2 * e + hh] * qfac, fmaf(kb[r], qs[nb][hh][r], v));
            v = ok ? v : -INFINITY;
            s[mt][nb][2 * e + hh] = v;
            up |= v > m[nb][hh] + kSlack;
          }
        }
      }
    }
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
    float vs[MT][2][NG];
    bool big = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int tk = 16 * mt + g + 8 * e;
        const bool ok = tk >= lo && tk < hi;
        float vb[NG];
        load_groups<E, NG>(vsc, tk, ok, vs[mt][e]);
        load_groups<E, NG>(vbi, tk, ok, vb);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const float pr = exp2_from(s[mt][nb][2 * e + hh], m[nb][hh]);
            s[mt][nb][2 * e + hh] = pr;
            l[nb][hh] += pr;
#pragma unroll
            for (int r = 0; r < NG; ++r) ob[nb][hh][r] = fmaf(pr, vb[r], ob[nb][hh][r]);
          }
        }
#pragma unroll
        for (int r = 0; r < NG; ++r) big |= fabsf(vs[mt][e][r]) > vlim[r];
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
          const float inv = ldexpf(1.0f, 6 - e);
          const float f = vlim[r] > 0.0f ? inv / vinv[r] : 1.0f;  // o is still zero the first time
          vinv[r] = inv;
          vlim[r] = ldexpf(1.0f, min(e + 8, 127));
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
        ldsm_x4_t(va.at(r0 + 16 * mt + 8 * (mq & 1) + r8, c + (mq >> 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < KPC; ++i) {
            const int k = (c + j) * KPC + i, r = k / 4;
            const uint32_t x0 = a[2 * j], x1 = a[2 * j + 1];
            uint32_t f0, f1, f2, f3;
            if constexpr (BITS == 8) {
              f0 = code_pair_u8(x0, 0x4240u), f1 = code_pair_u8(x0, 0x4341u);
              f2 = code_pair_u8(x1, 0x4240u), f3 = code_pair_u8(x1, 0x4341u);
            } else {
              f0 = code_pair_u4(x0, 2 * i), f1 = code_pair_u4(x0, 2 * i + 1);
              f2 = code_pair_u4(x1, 2 * i), f3 = code_pair_u4(x1, 2 * i + 1);
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
            w.o[hd * (D + 4) + d] = fmaf(o[nb][k][e], back, ob[nb][e][k / 4]);
            w.o[hd * (D + 4) + d + 1] = fmaf(o[nb][k][2 + e], back, ob[nb][e][k / 4]);
          }
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------
// fp32 pools (dense, or codes with fp32 scales) on the FMA pipes: the tensor
// cores have no fp32 product. q.k: a lane holds one token and every
// kParts-th 16-byte chunk of its row; p.v: a lane holds D / 32 dims and walks
// the tokens, p broadcast by shuffles. q (times scale * log2 e) and, for
// codes, its sum over each chunk lie in shared memory.
// ---------------------------------------------------------------------------
template <int BITS, int D, int NB>
struct FmaAttend {
  using F = PagedFmt<4, BITS, D>;
  static constexpr int GM = 8 * NB, NCH = F::kNChunk, EPC = F::kEpc, NG = F::kGroups;
  static constexpr int TW = F::kTile / kPagedWarps, PARTS = 32 / TW, DPL = D / 32;
  float m[GM], l[GM], o[GM][DPL];

  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[EPC]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < EPC; ++i) {
      if constexpr (BITS == 0) x[i] = __uint_as_float(u[i]);
      else if constexpr (BITS == 8) x[i] = float((u[i / 4] >> (8 * (i % 4))) & 255u);
      else x[i] = float((u[i / 8] >> (4 * (i % 8))) & 15u);
    }
  }

  // every consumer thread calls; qf: [G][D] then [G][NCH] chunk sums
  __device__ __forceinline__ void begin(const PagedParams& p, float* qf, int b, int h, int warp, int lane) {
    const float* q = static_cast<const float*>(p.q) + (int64_t(b) * p.Hkv * p.G + int64_t(h) * p.G) * D;
    const int t = warp * 32 + lane;
    for (int i = t; i < p.G * D; i += 32 * kPagedWarps) qf[i] = __ldg(q + i) * p.scale_log2;
    if constexpr (BITS != 0) {
      for (int i = t; i < p.G * NCH; i += 32 * kPagedWarps) {
        float sum = 0.0f;
        for (int d = 0; d < EPC; ++d) sum += __ldg(q + (i / NCH) * D + (i % NCH) * EPC + d);
        qf[p.G * D + i] = sum * p.scale_log2;
      }
    }
    named_barrier(1, 32 * kPagedWarps);
#pragma unroll
    for (int g = 0; g < GM; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.0f;
#pragma unroll
      for (int i = 0; i < DPL; ++i) o[g][i] = 0.0f;
    }
  }

  __device__ __forceinline__ void tile(const PagedParams& p, const float* qf, const TileView& t, int warp, int lane) {
    const int tok = lane % TW, part = lane / TW, r0 = warp * TW;
    const int lo = max(t.lo - r0, 0), hi = min(t.hi - r0, TW);
    if (hi <= lo) return;
    const TileAddr<F> ka{smem_u32(t.stage), t.pb_log}, va{smem_u32(t.stage) + F::kKvBytes, t.pb_log};
    const float* ksc = reinterpret_cast<const float*>(t.stage + 2 * F::kKvBytes) + r0 * NG;
    const float *kbi = ksc + F::kTile * NG, *vsc = ksc + 2 * F::kTile * NG, *vbi = ksc + 3 * F::kTile * NG;
    const bool ok = tok >= lo && tok < hi;
    float s[GM];
#pragma unroll
    for (int g = 0; g < GM; ++g) s[g] = 0.0f;
#pragma unroll 2
    for (int c = part; c < NCH; c += PARTS) {
      float x[EPC];
      unpack(lds128(ka.at(r0 + tok, c)), x);
      float sc = 1.0f, bi = 0.0f;
      if constexpr (BITS != 0) {
        sc = ksc[tok * NG + c * EPC / 64];
        bi = kbi[tok * NG + c * EPC / 64];
      }
#pragma unroll
      for (int g = 0; g < GM; ++g) {
        if (g < p.G) {
          const float4* qv = reinterpret_cast<const float4*>(qf + g * D + c * EPC);
          float a = 0.0f;
#pragma unroll
          for (int i = 0; i < EPC; i += 4) {
            const float4 w = qv[i / 4];
            a = fmaf(w.x, x[i], a);
            a = fmaf(w.y, x[i + 1], a);
            a = fmaf(w.z, x[i + 2], a);
            a = fmaf(w.w, x[i + 3], a);
          }
          if constexpr (BITS != 0) s[g] = fmaf(sc, a, fmaf(bi, qf[p.G * D + g * NCH + c], s[g]));
          else s[g] += a;
        }
      }
    }
    bool up = false;
#pragma unroll
    for (int g = 0; g < GM; ++g) {
      if (g < p.G) {
#pragma unroll
        for (int x = TW; x < 32; x <<= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], x);
        s[g] = ok ? s[g] : -INFINITY;
        up |= s[g] > m[g] + kSlack;
      }
    }
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int g = 0; g < GM; ++g) {
        if (g < p.G) {
          const float f = raise_max(m[g], warp_max(s[g]));
          l[g] *= f;
#pragma unroll
          for (int i = 0; i < DPL; ++i) o[g][i] *= f;
        }
      }
    }
#pragma unroll
    for (int g = 0; g < GM; ++g) {
      if (g < p.G) {
        s[g] = exp2_from(s[g], m[g]);
        if (part == 0) l[g] += s[g];
      }
    }
#pragma unroll 2
    for (int tk = lo; tk < hi; ++tk) {
      float v[DPL];
      constexpr int BPL = F::kRowBytes / 32;  // bytes of a row that a lane owns
      const uint32_t a = va.at(r0 + tk, lane * BPL / 16) + (lane * BPL) % 16;
      if constexpr (BITS == 0) {
        if constexpr (DPL == 4) {
          const float4 f = lds_f4(a);
          v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
          const uint2 f = lds64(a);
          v[0] = __uint_as_float(f.x), v[1] = __uint_as_float(f.y);
        }
      } else {
        const uint32_t w = lds32(a & ~3u) >> (8 * (a & 3u));
        const float sc = vsc[tk * NG + lane * DPL / 64], bi = vbi[tk * NG + lane * DPL / 64];
#pragma unroll
        for (int i = 0; i < DPL; ++i) v[i] = fmaf(sc, float((w >> (BITS * i)) & ((1u << BITS) - 1u)), bi);
      }
#pragma unroll
      for (int g = 0; g < GM; ++g) {
        if (g < p.G) {
          const float pr = __shfl_sync(0xffffffffu, s[g], tk);
#pragma unroll
          for (int i = 0; i < DPL; ++i) o[g][i] = fmaf(pr, v[i], o[g][i]);
        }
      }
    }
  }

  __device__ __forceinline__ void end(const PagedParams& p, const WarpPart<D>& w, int lane) {
#pragma unroll
    for (int g = 0; g < GM; ++g) {
      if (g < p.G) {
        const float ls = warp_sum(l[g]);
        if (lane == 0) {
          w.ml[2 * g] = m[g];
          w.ml[2 * g + 1] = ls;
        }
#pragma unroll
        for (int i = 0; i < DPL; ++i) w.o[g * (D + 4) + lane * DPL + i] = o[g][i];
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
  const int raw = __ldg(p.lengths + b);
  if ((raw < 0 || raw > cap) && p.flags && blockIdx.x == 0) atomicOr(p.flags, kErrBadIndex);
  const int len = raw < 0 ? 0 : raw > cap ? int(cap) : raw;
  return {p.window > 0 && len > p.window ? len - p.window : 0, len};
}
__device__ __forceinline__ int tiles_of(TokenRange r, int tile) {
  return r.end > r.begin ? (r.end + tile - 1) / tile - r.begin / tile : 0;
}

// The line of U units (tile, pair) in equal pieces for the CTAs that take
// part, at least min_tiles each: the first `rem` pieces have base + 1 units.
struct Pieces {
  int n, base, rem;
  __device__ __forceinline__ Pieces(const PagedParams& p, int U) {
    n = min((U + p.min_tiles - 1) / p.min_tiles, p.ncta);
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
    if (u >= u1) return false;
    while (prefix[b + 1] * Hkv <= u) ++b;  // ends: u < prefix[B] * Hkv
    s.b = b;
    s.nt = prefix[b + 1] - prefix[b];
    const int r = u - prefix[b] * Hkv;
    s.h = r / s.nt;
    s.i0 = r - s.h * s.nt;
    s.i1 = min(s.nt, s.i0 + u1 - u);
    u += s.i1 - s.i0;
    return true;
  }
};

template <typename E, int BITS, int D, int NB, bool kTensor>
struct PickAttend;
template <typename E, int D, int NB>
struct PickAttend<E, 0, D, NB, true> { using type = DenseAttend<E, D, NB>; };
template <typename E, int BITS, int D, int NB>
struct PickAttend<E, BITS, D, NB, true> { using type = CodesAttend<E, BITS, D, NB>; };
template <typename E, int BITS, int D, int NB>
struct PickAttend<E, BITS, D, NB, false> { using type = FmaAttend<BITS, D, NB>; };

// The producer warp: this CTA's tiles into the ring, stage by stage.
template <typename E, int BITS, int D>
__device__ __forceinline__ void paged_produce(const PagedParams& p, const CUtensorMap* tmK, const CUtensorMap* tmV,
                                              uint8_t* ring, uint64_t* full, uint64_t* empty, Walk walk, int lane) {
  using F = PagedFmt<sizeof(E), BITS, D>;
  const uint64_t pol = stream_policy(false);
  const int pb = min(p.P, F::kTile), nb = F::kTile / pb;   // rows per box, boxes per tile
  const int p_log = __ffs(p.P) - 1, pb_log = __ffs(pb) - 1;
  const int oob_row = int(p.n_pages * p.Hkv * p.P);  // past the tensor: TMA fills zeros
  int it = 0;
  Segment s;
  while (walk.next(s)) {
    const TokenRange r = token_range(p, s.b);
    const int* row = p.tables + int64_t(s.b) * p.W;
    const int t0 = r.begin / F::kTile;
    const int last_slot = (r.end - 1) >> p_log, first_slot = r.begin >> p_log;
    auto load = [&](int slot) { return slot >= first_slot && slot <= last_slot ? __ldg(row + slot) : -1; };
    int base = ((t0 + s.i0) * F::kTile) >> p_log;
    int cur = load(base + lane), nxt = load(base + 32 + lane);
    for (int i = s.i0; i < s.i1; ++i, ++it) {
      const int st = it % p.stages, tok = (t0 + i) * F::kTile;
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
      if (it >= p.stages && !mbar_wait(empty + st, uint32_t(it / p.stages - 1) & 1u, p.flags)) {
        // the consumers gave up: no more copies, but those under way must land before this CTA may end
        for (int k = max(0, it - p.stages); k < it; ++k) mbar_wait(full + k % p.stages, uint32_t(k / p.stages) & 1u, nullptr);
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
  __shared__ int warp_tot[kPagedThreads / 32];
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
  griddep_launch_dependents();
  griddep_wait();

  // tiles before each sequence
  const int per = (p.B + kPagedThreads - 1) / kPagedThreads;
  int mine = 0;
  for (int k = 0; k < per; ++k) {
    const int b = tid * per + k;
    if (b < p.B) mine += tiles_of(token_range(p, b), F::kTile);
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
      if (blockIdx.x == 0) p.prefix[b] = run;
      run += tiles_of(token_range(p, b), F::kTile);
      if (b == p.B - 1) {
        prefix[p.B] = run;
        if (blockIdx.x == 0) p.prefix[p.B] = run;
      }
    }
  }
  __syncthreads();

  const Pieces pieces(p, prefix[p.B] * p.Hkv);
  if (int(blockIdx.x) >= pieces.n) return;
  Walk walk(prefix, p.B, p.Hkv, pieces.begin(blockIdx.x), pieces.begin(blockIdx.x + 1));

  if (warp == kPagedWarps) {
    paged_produce<E, BITS, D>(p, &tmK, &tmV, sm, full, empty, walk, lane);
    return;
  }
  using A = typename PickAttend<E, BITS, D, NB, F::kTensor>::type;
  const int pb_log = __ffs(min(p.P, F::kTile)) - 1;
  A att;
  Segment s;
  int it = 0;
  bool dead = false, first = true;
  while (walk.next(s)) {
    const TokenRange r = token_range(p, s.b);
    const int t0 = r.begin / F::kTile;
    att.begin(p, qf, s.b, s.h, warp, lane);
    for (int i = s.i0; i < s.i1; ++i, ++it) {
      const int st = it % p.stages, tok = (t0 + i) * F::kTile;
      if (!dead) dead = !mbar_wait(full + st, uint32_t(it / p.stages) & 1u, p.flags);
      if (!dead) {
        att.tile(p, qf, TileView{sm + st * F::kStageBytes, pb_log, r.begin - tok, r.end - tok}, warp, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + st);
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
        if (p.sinks) L += exp2f(fmaf(__ldg(p.sinks + hq), 1.4426950408889634f, -(M == -INFINITY ? 0.0f : M)));
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
  // after a wait that expired: copies under way still land in this CTA's memory
  if (dead)
    for (int k = max(0, it - p.stages); k < it; ++k) mbar_wait(full + k % p.stages, uint32_t(k / p.stages) & 1u, nullptr);
}

// Joins the segments of one query head (grid: B * Hq blocks) in a fixed
// order; a pair that one CTA did alone is already written, an empty one is
// written here as zeros. Bound by the latency of its dependent loads, not by
// their bytes (a few MB at most, from L2): warp w takes the segments w, w + 8,
// ..., each lane first the (m, l) of one of them, and the o rows are loaded
// eight at a time, the first eight before the weights are known.
template <typename E, int D>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const __grid_constant__ PagedParams p) {
  constexpr int NW = kMergeThreads / 32, V = D / 32, BATCH = 8;
  __shared__ float red[NW][D], top[NW], tot[NW];
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Hq = p.Hkv * p.G, b = blockIdx.x / Hq, hq = blockIdx.x % Hq, h = hq / p.G, g = hq % p.G;
  const int pre = p.prefix[b], nt = p.prefix[b + 1] - pre, all = p.prefix[p.B];
  E* out = static_cast<E*>(p.out) + int64_t(blockIdx.x) * D;
  if (nt == 0) {
    for (int d = tid; d < D; d += kMergeThreads) out[d] = Elt<E>::from_f32(0.0f);
    return;
  }
  const Pieces pieces(p, all * p.Hkv);
  const int a = pre * p.Hkv + h * nt;  // the pair's first unit
  const int c0 = pieces.of(a), c1 = pieces.of(a + nt - 1), ns = c1 - c0 + 1;
  if (ns == 1) return;
  const int stride = paged_part_floats(p.G, D);
  // a CTA leaves its first segment in slot 0: the pair is that for all but, perhaps, c0
  const int skip = pieces.begin(c0) < a ? 1 : 0;
  auto slot = [&](int i) { return p.part + (int64_t(c0 + i) * 2 + (i == 0 ? skip : 0)) * stride; };
  float M = -INFINITY, L = 0.0f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  for (int base = warp; base < ns; base += 32 * NW) {  // lane j: segment base + j * NW
    const int n = min(32, (ns - base + NW - 1) / NW);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < n) ml = *reinterpret_cast<const float2*>(slot(base + lane * NW) + p.G * D + 2 * g);
    float x[BATCH][V];
    auto load = [&](int j0) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        if (j0 + j < n) {
          const float* o = slot(base + (j0 + j) * NW) + g * D + lane * V;
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
#pragma unroll
  for (int i = 0; i < V; ++i) red[warp][lane * V + i] = acc[i];
  if (lane == 0) {
    top[warp] = M;
    tot[warp] = L;
  }
  __syncthreads();
  if (tid >= D) return;
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
  if (p.sinks) L += exp2f(fmaf(__ldg(p.sinks + hq), 1.4426950408889634f, -(M == -INFINITY ? 0.0f : M)));
  out[tid] = Elt<E>::from_f32(L == 0.0f ? 0.0f : O / L);
}

}  // namespace sd
