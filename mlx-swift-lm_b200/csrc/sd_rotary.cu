// sd_rotary.cu -- per-head RMS norm and rotary positions of queries and keys,
// alone or with the keys and values stored into the pages of a KV pool, and
// copies of whole pages.
//
// Rotation, for a row x of head_dim elements at position pos:
//   y = x * rsqrt(mean(x^2) + eps) * w                        (if a norm is given)
//   (a, b) -> factor * (a cos - b sin, b cos + a sin), angle pos * inv_freq[i],
//   where pair i is (y[i], y[i + rot/2]), or (y[2i], y[2i + 1]) in the
//   traditional layout; elements from rot on pass through.
// Every row is read and written once, and that traffic bounds the call: about
// 10 operations per element. All of it is fp32 with one rounding at the end.
// The angle is reduced in fp64: pos * inv_freq / (2 pi) loses no more than
// 2^-53 of itself, so positions of a million are as exact as small ones,
// where an fp32 product would be off by 0.03 rad.
#include <cuda_runtime.h>

#include "sd_paged.h"
#include "sd_update.cuh"

namespace sd {

namespace {

// 16-byte (or narrower) register chunk of V elements.
template <int BYTES> struct Chunk;
template <> struct Chunk<16> { using T = uint4; };
template <> struct Chunk<8> { using T = uint2; };
template <> struct Chunk<4> { using T = uint32_t; };
template <> struct Chunk<2> { using T = uint16_t; };

template <typename E, int V> union Pack {
  typename Chunk<V * sizeof(E)>::T raw;
  E e[V];
  __device__ Pack() {}
};


}  // namespace

// One group of lanes per row; a lane holds chunk pairs of V elements: pair j
// is the elements [jV, jV + V) of the first rotated half and the same of the
// second, or 2V neighbours (traditional layout, and past the rotated part).
// So a lane always holds both elements of a rotation and needs no exchange.
// A block takes kRotUnroll rows per group, consecutive in (token, head)
// order, loads them all first, and while they are under way puts cos and sin
// of its few tokens into shared memory: one sincos per token and pair instead
// of one per row. BITS 4 / 8: k and v rows are rounded to E, staged in shared
// memory and quantized from there a warp per row.
template <typename E, int V, int BITS>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int CPL = V >= 4 ? 1 : V == 2 ? 2 : 4;  // chunk pairs per lane for head_dim up to 256
  using P = Pack<E, V>;
  extern __shared__ float smem[];
  float* cs = smem;                                  // [span][2][rot2]
  float* wn = cs + int64_t(p.span) * 2 * p.rot2;     // [2][D] norm weights
  E* stage = reinterpret_cast<E*>(smem + rotary_stage_at(p.span, p.rot2, p.D));  // [rows per block][D] (BITS)
  const int D = p.D, pairs = D / (2 * V), lg_log = rotary_lanes_log(D, V), lg = 1 << lg_log;
  const int groups = kRotThreads >> lg_log, rows = groups * kRotUnroll;
  const int tid = threadIdx.x, sub = tid & (lg - 1), grp = tid >> lg_log;
  griddep_launch_dependents();
  griddep_wait();

  const int64_t task0 = int64_t(blockIdx.x) * rows;
  const int64_t n0 = task0 / p.R;
  const int rem0 = int(task0 - n0 * p.R);
  const int half = p.traditional ? 0 : p.rot2 / V;   // chunk pairs that straddle the two halves

  // Element offset of chunk i (0, 1) of pair j.
  auto place = [&](int j, int i) { return j < half ? j * V + i * p.rot2 : 2 * j * V + i * V; };

  P x[kRotUnroll][CPL][2];
#pragma unroll
  for (int u = 0; u < kRotUnroll; ++u) {
    const int local = u * groups + grp;
    if (task0 + local >= p.tasks) continue;
    const int k = (rem0 + local) / p.R, r = rem0 + local - k * p.R;
    const int64_t n = n0 + k;
    const int64_t bt = n / p.L, t = n - bt * p.L;
    const Rows& s = r < p.Hq ? p.q : r < p.Hq + p.Hkv ? p.k : p.v;
    const int hd = r < p.Hq ? r : r < p.Hq + p.Hkv ? r - p.Hq : r - p.Hq - p.Hkv;
    const E* src = static_cast<const E*>(s.data) + bt * s.batch + t * s.token + hd * s.head;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int j = c * lg + sub;
      if (j < pairs) {
        x[u][c][0].raw = *reinterpret_cast<const decltype(P::raw)*>(src + place(j, 0));
        x[u][c][1].raw = *reinterpret_cast<const decltype(P::raw)*>(src + place(j, 1));
      }
    }
  }

  if (p.rot2) {
    const int64_t last = min(task0 + rows, p.tasks) - 1;
    const int span = int(last / p.R - n0) + 1;
    for (int i = tid; i < span * p.rot2; i += kRotThreads) {
      const int k = i / p.rot2, f = i - k * p.rot2;
      // turns of the angle, less whole turns
      double turns = double(__ldg(p.positions + n0 + k)) * (double(__ldg(p.inv_freq + f)) * 0.15915494309189535);
      turns -= rint(turns);
      float sn, c;
      sincospif(2.0f * float(turns), &sn, &c);
      cs[(2 * k) * p.rot2 + f] = c * p.factor;
      cs[(2 * k + 1) * p.rot2 + f] = sn * p.factor;
    }
  }
  if (p.q_norm)
    for (int i = tid; i < D; i += kRotThreads) wn[i] = Elt<E>::to_f32(static_cast<const E*>(p.q_norm)[i]);
  if (p.k_norm)
    for (int i = tid; i < D; i += kRotThreads) wn[D + i] = Elt<E>::to_f32(static_cast<const E*>(p.k_norm)[i]);
  __syncthreads();

#pragma unroll
  for (int u = 0; u < kRotUnroll; ++u) {
    const int local = u * groups + grp;
    const bool live = task0 + local < p.tasks;
    const int k = (rem0 + local) / p.R, r = rem0 + local - k * p.R;
    const int64_t n = n0 + k;
    const bool is_q = r < p.Hq, is_v = r >= p.Hq + p.Hkv;
    const int hd = is_q ? r : is_v ? r - p.Hq - p.Hkv : r - p.Hq;
    float f[CPL][2][V];
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) f[c][i][e] = live && c * lg + sub < pairs ? Elt<E>::to_f32(x[u][c][i].e[e]) : 0.0f;
    if (p.q_norm || p.k_norm) {  // every lane of the warp takes part in the shuffles
      float sq = 0.0f;
#pragma unroll
      for (int c = 0; c < CPL; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) sq = fmaf(f[c][i][e], f[c][i][e], sq);
      for (int o = 1; o < lg; o <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      if (!is_v && (is_q ? p.q_norm : p.k_norm)) {
        const float inv = rsqrtf(sq / float(D) + p.eps);
        const float* w = wn + (is_q ? 0 : D);
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const int j = c * lg + sub;
          if (j < pairs) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < V; ++e) f[c][i][e] *= inv * w[place(j, i) + e];
          }
        }
      }
    }
    if (!live) continue;
    if (!is_v && p.rot2) {
      const float *co = cs + 2 * k * p.rot2, *si = co + p.rot2;
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const int j = c * lg + sub;
        if (j < pairs) {
          if (p.traditional) {
            // the 2V neighbours are V whole pairs
            float z[2 * V];
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = f[c][0][e], z[V + e] = f[c][1][e];
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const int i = j * V + e;
              if (i < p.rot2) {
                const float a = z[2 * e], b = z[2 * e + 1];
                z[2 * e] = fmaf(a, co[i], -b * si[i]);
                z[2 * e + 1] = fmaf(b, co[i], a * si[i]);
              }
            }
#pragma unroll
            for (int e = 0; e < V; ++e) f[c][0][e] = z[e], f[c][1][e] = z[V + e];
          } else if (j < half) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float a = f[c][0][e], b = f[c][1][e];
              f[c][0][e] = fmaf(a, co[j * V + e], -b * si[j * V + e]);
              f[c][1][e] = fmaf(b, co[j * V + e], a * si[j * V + e]);
            }
          }
        }
      }
    }
    // where the row goes
    E* dst = nullptr;
    if (is_q || !p.tables) {
      const Rows& o = is_q ? p.q_out : p.k_out;
      const int64_t bt = n / p.L, t = n - bt * p.L;
      dst = static_cast<E*>(o.data) + bt * o.batch + t * o.token + hd * o.head;
    } else if (BITS != 0) {
      dst = stage + local * D;
    } else {
      const int pos = __ldg(p.positions + n), sq = p.seq ? __ldg(p.seq + n) : int(n);
      if (pos >= 0) {
        const int slot = pos >> p.page_shift;
        const int page = sq >= 0 && sq < p.B && slot < p.W ? __ldg(p.tables + int64_t(sq) * p.W + slot) : -1;
        if (page >= 0 && page < p.n_pages) {
          dst = static_cast<E*>(is_v ? p.v_data : p.k_data) +
                ((int64_t(page) * p.Hkv + hd) * p.P + (pos & (p.P - 1))) * D;
        } else if (p.flags) {
          atomicOr(p.flags, kErrBadIndex);
        }
      }
    }
    if (dst) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const int j = c * lg + sub;
        if (j < pairs) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            P y;
#pragma unroll
            for (int e = 0; e < V; ++e) y.e[e] = is_v ? x[u][c][i].e[e] : Elt<E>::from_f32(f[c][i][e]);
            *reinterpret_cast<decltype(P::raw)*>(dst + place(j, i)) = y.raw;
          }
        }
      }
    }
  }

  if constexpr (BITS != 0) {
    __syncthreads();
    const int warp = tid >> 5, lane = tid & 31, NG = D / 64, words = D * BITS / 32;
    for (int local = warp; local < rows && task0 + local < p.tasks; local += kRotThreads / 32) {
      const int k = (rem0 + local) / p.R, r = rem0 + local - k * p.R;
      if (r < p.Hq) continue;
      const int64_t n = n0 + k;
      const int pos = __ldg(p.positions + n), sq = p.seq ? __ldg(p.seq + n) : int(n);
      if (pos < 0) continue;
      const int slot = pos >> p.page_shift;
      const int page = sq >= 0 && sq < p.B && slot < p.W ? __ldg(p.tables + int64_t(sq) * p.W + slot) : -1;
      if (page < 0 || page >= p.n_pages) {
        if (p.flags && lane == 0) atomicOr(p.flags, kErrBadIndex);
        continue;
      }
      const bool is_v = r >= p.Hq + p.Hkv;
      const int hd = is_v ? r - p.Hq - p.Hkv : r - p.Hq;
      const int64_t row = (int64_t(page) * p.Hkv + hd) * p.P + (pos & (p.P - 1));
      uint32_t* wq = static_cast<uint32_t*>(is_v ? p.v_data : p.k_data) + row * words;
      E* sc = static_cast<E*>(is_v ? p.v_scales : p.k_scales) + row * NG;
      E* bi = static_cast<E*>(is_v ? p.v_biases : p.k_biases) + row * NG;
      const E* src = stage + local * D;
      if (D == 128) quantize_row_warp<E, BITS, 128>(src, wq, sc, bi, lane);
      else quantize_row_warp<E, BITS, 64>(src, wq, sc, bi, lane);
    }
  }
}

template <typename E, int BITS>
static const void* rotary_pick(int vec) {
  switch (vec) {
    case 8:
      if constexpr (sizeof(E) == 2) return reinterpret_cast<const void*>(&rotary_kernel<E, 8, BITS>);
      return nullptr;
    case 4: return reinterpret_cast<const void*>(&rotary_kernel<E, 4, BITS>);
    case 2: return reinterpret_cast<const void*>(&rotary_kernel<E, 2, BITS>);
    case 1: return reinterpret_cast<const void*>(&rotary_kernel<E, 1, BITS>);
    default: return nullptr;
  }
}
template <typename E>
static const void* rotary_bits(int bits, int vec) {
  return bits == 0 ? rotary_pick<E, 0>(vec) : bits == 4 ? rotary_pick<E, 4>(vec) : rotary_pick<E, 8>(vec);
}

const void* rotary_kernel_for(int dtype, int bits, int vec) {
  return dtype == 0 ? rotary_bits<float>(bits, vec) : dtype == 1 ? rotary_bits<__half>(bits, vec)
                                                                 : rotary_bits<__nv_bfloat16>(bits, vec);
}

// Page dst[i] = page src[i] in every array and layer: a pure copy, bound by
// HBM (every byte read once and written once). Pages are contiguous in each
// array, so the work is cut into pieces of at most kCopyPiece bytes; a block
// moves one piece with four 16-byte loads per thread in flight.
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  griddep_launch_dependents();
  griddep_wait();
  for (int64_t w = blockIdx.x; w < p.total; w += gridDim.x) {
    const int64_t unit = w / p.per_pair;           // (layer, pair)
    int piece = int(w - unit * p.per_pair);
    const int64_t layer = unit / p.n;
    const int i = int(unit - layer * p.n);
    const int src = __ldg(p.src + i), dst = __ldg(p.dst + i);
    if (src < 0 || src >= p.n_pages || dst < 0 || dst >= p.n_pages) {
      if (p.flags && threadIdx.x == 0) atomicOr(p.flags, kErrBadIndex);
      continue;
    }
    int a = 0;
    while (piece >= p.pieces[a]) piece -= p.pieces[a++];
    const int64_t page = p.bytes[a], at = int64_t(piece) * kCopyPiece;
    const int n16 = int(min(int64_t(kCopyPiece), page - at) / 16);
    const uint4* s = reinterpret_cast<const uint4*>(p.array[a] + (layer * p.n_pages + src) * page + at);
    uint4* d = reinterpret_cast<uint4*>(p.array[a] + (layer * p.n_pages + dst) * page + at);
    constexpr int K = kCopyPiece / 16 / kCopyThreads;
    uint4 v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int x = k * kCopyThreads + threadIdx.x;
      if (x < n16) v[k] = __ldcs(s + x);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int x = k * kCopyThreads + threadIdx.x;
      if (x < n16) __stcs(d + x, v[k]);
    }
  }
}

const void* copy_pages_kernel_ptr() { return reinterpret_cast<const void*>(&copy_pages_kernel); }

}  // namespace sd
