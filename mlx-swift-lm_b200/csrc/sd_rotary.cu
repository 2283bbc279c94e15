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
  uint32_t word[V * sizeof(E) / 4 ? V * sizeof(E) / 4 : 1];
  __device__ Pack() {}
  __device__ __forceinline__ void zero() { memset(&raw, 0, sizeof(raw)); }
  __device__ __forceinline__ void unpack(float* f) const {
    if constexpr (sizeof(E) == 2 && V >= 2) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) unpack_word<E>(word[i], f + 2 * i);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = Elt<E>::to_f32(e[i]);
    }
  }
  __device__ __forceinline__ void pack(const float* f) {
    if constexpr (sizeof(E) == 2 && V >= 2) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) word[i] = pack2<E>(f[2 * i], f[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = Elt<E>::from_f32(f[i]);
    }
  }
};

// Copy one chunk to shared memory, asynchronously where its size allows.
template <int BYTES>
__device__ __forceinline__ void copy_chunk(void* dst, const void* src) {
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  } else if constexpr (BYTES >= 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
  } else {
    *static_cast<uint16_t*>(dst) = *static_cast<const uint16_t*>(src);
  }
}

// Quantize elements [sub * EL, sub * EL + EL) of a row of E whose lanes hold EL
// elements each, with the affine group-64 rule and the fp32 operations of
// quantize_row_regs; every lane of the warp calls, `live` ones store.
template <typename E, int BITS, int EL>
__device__ __forceinline__ void quantize_part(const E* row, uint8_t* wq, E* sc, E* bi, int sub, bool live) {
  constexpr int LPG = 64 / EL;  // lanes per quantization group
  const float n_bins = float((1 << BITS) - 1);
  float w[EL];
#pragma unroll
  for (int e = 0; e < EL; ++e) w[e] = Elt<E>::to_f32(row[sub * EL + e]);
  float wmax = w[0], wmin = w[0];
#pragma unroll
  for (int e = 1; e < EL; ++e) wmax = fmaxf(wmax, w[e]), wmin = fminf(wmin, w[e]);
#pragma unroll
  for (int o = 1; o < LPG; o <<= 1) {
    wmax = fmaxf(wmax, __shfl_xor_sync(0xffffffffu, wmax, o));
    wmin = fminf(wmin, __shfl_xor_sync(0xffffffffu, wmin, o));
  }
  float scale = fmaxf(__fdiv_rn(__fsub_rn(wmax, wmin), n_bins), 1e-7f);
  const bool low = fabsf(wmin) > fabsf(wmax);
  if (!low) scale = -scale;
  const float edge = low ? wmin : wmax;
  const float q0 = rintf(__fdiv_rn(edge, scale));
  if (q0 != 0.0f) scale = __fdiv_rn(edge, q0);
  const float bias = q0 == 0.0f ? 0.0f : edge;
  constexpr int BYTES = EL * BITS / 8;
  uint32_t words[(BYTES + 3) / 4] = {};
#pragma unroll
  for (int e = 0; e < EL; ++e) {
    float c = rintf(__fdiv_rn(__fsub_rn(w[e], bias), scale));
    c = fminf(fmaxf(c, 0.0f), n_bins);
    words[e * BITS / 32] |= uint32_t(c) << (e * BITS % 32);
  }
  if (!live) return;
  uint8_t* d = wq + sub * BYTES;
  if constexpr (BYTES == 16) *reinterpret_cast<uint4*>(d) = make_uint4(words[0], words[1], words[2], words[3]);
  else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(d) = make_uint2(words[0], words[1]);
  else if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(d) = words[0];
  else if constexpr (BYTES == 2) *reinterpret_cast<uint16_t*>(d) = uint16_t(words[0]);
  else *d = uint8_t(words[0]);
  if (sub % LPG == 0) {
    sc[sub / LPG] = Elt<E>::from_f32(scale);
    bi[sub / LPG] = Elt<E>::from_f32(bias);
  }
}

}  // namespace

// Which elements a lane holds, and where it finds the other one of a rotation.
enum RotaryForm {
  kHalves,   // chunk pair j: [jV, jV + V) of both rotated halves, so every rotation is within a lane
  kNearby,   // traditional layout: two chunks that are half a row apart, each of whole rotations
  kShifted,  // halves that are no whole number of chunks: as kNearby, the other elements from shared memory
};

// A warp takes rows of one kind (query, key or value) and of few tokens: a
// group of lanes holds one row at a time and stays with one token, so what
// depends on the position and the weights is computed once and stays in
// registers. With the norm's weights w folded into cos and sin, a rotation is
//   a' = inv * (a (w_a cos) - b (w_b sin)),  b' = inv * (b (w_b cos) + a (w_a sin)),
// inv = the row's 1 / rms. A lane holds chunk pairs of V elements (RotaryForm);
// the lanes' first chunks lie side by side, and so do their second ones, as an
// access that skips every other 16 bytes moves half as much (traditional
// layout with neighbouring chunks 38 us instead of 27 at 6023 tokens of 48
// heads). Rows are copied kRotDepth passes ahead into shared memory (each lane
// its own chunks, so nothing waits for another lane but in kShifted); while the
// first are under way the warp computes its tokens' cos and sin, one pair per
// lane, and exchanges them through shared memory. No barrier wider than a warp.
// BITS 4 / 8: key and value rows are rounded to E, staged in shared memory and
// quantized from there by the group of lanes that holds the row.
// CPL: chunk pairs per lane.
// Measured, bf16 rows of 128 with norms: 32K tokens of 40 heads (671 MB) 107.5
// us, 6.2 TB/s; 6023 tokens of 48 heads (148 MB, floor 22.6 us) 27.5 us in the
// half layout, 27.6 traditional, 62 in kShifted.
template <typename E, int V, int CPL, int BITS, RotaryForm FORM>
__global__ void __launch_bounds__(kRotThreads, 5) rotary_kernel(const __grid_constant__ RotaryParams p) {
  static_assert(FORM != kShifted || CPL == 1, "one chunk pair per lane");
  using P = Pack<E, V>;
  extern __shared__ __align__(16) float smem[];
  const int D = p.D, pairs = D / (2 * V), lg_log = rotary_lanes_log(D, V), lg = 1 << lg_log;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (lg - 1), grp = lane >> lg_log;
  const int groups = 32 >> lg_log, pitch = rotary_pitch(p.rot2);
  float* cs = smem + warp * groups * 2 * pitch;      // [tokens of this warp][cos, sin]
  E* stage = reinterpret_cast<E*>(smem + kRotThreads / 32 * groups * 2 * pitch) + warp * groups * D;
  griddep_wait();
  griddep_launch_dependents();

  const int unit = blockIdx.x * (kRotThreads / 32) + warp;
  if (unit >= p.units) return;
  const bool is_v = unit >= p.kind[2].first, is_q = unit < p.kind[1].first;
  const RotaryParams::Kind& kd_ = p.kind[is_q ? 0 : is_v ? 2 : 1];
  const Rows& in = is_q ? p.q : is_v ? p.v : p.k;
  const int heads = is_q ? p.Hq : is_v ? p.Hv : p.Hkv;
  const int chunk = kd_.per(unit - kd_.first), first_pass = (unit - kd_.first - chunk * kd_.per.d) * kd_.span;
  // group g: token g mod 2^tok_log of the chunk, heads g / 2^tok_log, + step, ...
  const int tl = kd_.tok_log, step = groups >> tl, n0 = chunk << tl;
  const int n = n0 + (grp & ((1 << tl) - 1));
  const bool here = n < p.n_tokens;
  const int bt = p.L(n), tk = n - bt * p.L.d;
  const int half = FORM == kHalves ? p.rot2 / V : 0;  // chunk pairs of the two rotated halves
  // Element offset of chunk i (0, 1) of pair j.
  auto place = [&](int j, int i) {
    if constexpr (FORM == kHalves) return j < half ? j * V + i * p.rot2 : 2 * p.rot2 + (j - half) * V + i * (D / 2 - p.rot2);
    else if constexpr (V == 1) return 2 * j + i;
    else return j * V + i * (D / 2);
  };
  int at[CPL][2];
#pragma unroll
  for (int c = 0; c < CPL; ++c) at[c][0] = place(c * lg + sub, 0), at[c][1] = place(c * lg + sub, 1);
  const E* src = static_cast<const E*>(in.data) + bt * in.batch + tk * in.token;

  // where key and value rows go: a page slot (the same for every head), or k_out
  E* paged = nullptr;
  int64_t slot = -1;  // row of head 0; head h is h * P rows on
  bool store = here;
  if (!is_q && p.tables) {
    paged = static_cast<E*>(is_v ? p.v_data : p.k_data);
    const int pos = here ? p.positions[n] : -1, sq = here && p.seq ? p.seq[n] : n;
    store = pos >= 0;  // else padding
    if (store) {
      const int col = pos >> p.page_shift;
      const int page = sq >= 0 && sq < p.B && col < p.W ? p.tables[int64_t(sq) * p.W + col] : -1;
      if (page >= 0 && page < p.n_pages) {
        slot = int64_t(page) * p.Hkv * p.P + (pos & (p.P - 1));
      } else {
        store = false;
        if (p.flags && sub == 0) atomicOr(p.flags, kErrBadIndex);
      }
    }
  }
  const Rows& outr = is_q ? p.q_out : p.k_out;
  E* out = static_cast<E*>(outr.data) + bt * outr.batch + tk * outr.token;

  const E* w = is_v ? nullptr : static_cast<const E*>(is_q ? p.q_norm : p.k_norm);
  const int last = min(heads, (first_pass + kd_.span) * step);  // heads of this warp end here
  int hd = first_pass * step + (grp >> tl);
  // Rows under way, kRotDepth passes ahead. A lane's chunks lie together with the other lanes' (kShifted: as the row).
  constexpr int BYTES = V * int(sizeof(E)), PASS = CPL * 2 * 32 * BYTES;  // of one warp and pass
  uint8_t* ring = reinterpret_cast<uint8_t*>(smem) + p.ring_at + warp * kRotDepth * PASS +
                  (FORM == kShifted ? grp * D * int(sizeof(E)) : lane * BYTES);
  auto slot_of = [&](int st, int c, int i) {
    return ring + st * PASS + (FORM == kShifted ? at[c][i] * int(sizeof(E)) : (2 * c + i) * 32 * BYTES);
  };
  const E* from = src + hd * in.head;  // the row to load next
  const int64_t from_step = step * in.head;
  int ahead = hd;
  auto fetch = [&](int st) {
    if (here && ahead < last) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const int j = c * lg + sub;
        if (j < pairs) {
          copy_chunk<BYTES>(slot_of(st, c, 0), from + at[c][0]);
          copy_chunk<BYTES>(slot_of(st, c, 1), from + at[c][1]);
        }
      }
    }
    cp_async_commit();
    from += from_step;
    ahead += step;
  };
#pragma unroll
  for (int st = 0; st < kRotDepth; ++st) fetch(st);
  E* dst = BITS != 0 && paged ? stage + grp * D : paged ? paged + (slot + int64_t(hd) * p.P) * D : out + hd * outr.head;
  const int64_t dst_step = BITS != 0 && paged ? 0 : paged ? int64_t(step) * p.P * D : step * outr.head;

  // This lane's elements: own * k1 + other * k2, k1 = w_own cos, k2 = -w_other sin (first of a rotation) or w_other sin
  // (second). Bit e of `turned`: rotation e (kShifted: element e) is one; in kHalves a chunk pair is rotated all or not at all.
  float k1[CPL][2 * V], k2[CPL][2 * V];
  uint32_t turned[CPL], far[V];  // far: byte offsets within the row of the other elements, two to a word (kShifted)
  if (!is_v) {
    for (int i = lane; i < p.rot2 << tl; i += 32) {
      const int t = p.pairs(i), f = i - t * p.rot2;
      // turns of the angle, less whole turns
      const double pos = n0 + t < p.n_tokens ? double(p.positions[n0 + t]) : 0.0;
      double turns = pos * (double(p.inv_freq[f]) * 0.15915494309189535);
      turns -= rint(turns);
      float sn, c;
      sincospif(2.0f * float(turns), &sn, &c);
      cs[2 * t * pitch + f] = c * p.factor;
      cs[(2 * t + 1) * pitch + f] = sn * p.factor;
    }
    __syncwarp();
    const float* co_row = cs + 2 * (n - n0) * pitch;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int j = c * lg + sub;
      turned[c] = 0;
      float wt[2 * V];
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) wt[e] = 1.0f;
      if (w && j < pairs) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) wt[e] = Elt<E>::to_f32(w[at[c][e / V] + e % V]);
      }
      if constexpr (FORM != kShifted) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int a = FORM == kNearby ? 2 * e : e, b = FORM == kNearby ? 2 * e + 1 : V + e;
          const int f = FORM == kNearby ? (at[c][a / V] + a % V) / 2 : j * V + e;
          const bool turn = FORM == kHalves ? j < half : j < pairs && f < p.rot2;
          const float co = turn ? co_row[f] : 1.0f, si = turn ? co_row[pitch + f] : 0.0f;
          k1[c][a] = wt[a] * co;
          k1[c][b] = wt[b] * co;
          k2[c][a] = -(wt[b] * si);
          k2[c][b] = wt[a] * si;
          turned[c] |= uint32_t(turn) << e;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          const int x = at[c][e / V] + e % V, f = x < p.rot2 ? x : x - p.rot2;
          const bool turn = j < pairs && f < p.rot2;
          const int y = !turn ? 0 : x < p.rot2 ? x + p.rot2 : f;
          const float co = turn ? co_row[f] : 1.0f, si = turn ? co_row[pitch + f] : 0.0f;
          const float other = w && turn ? Elt<E>::to_f32(w[y]) : 1.0f;
          k1[c][e] = wt[e] * co;
          k2[c][e] = other * (x < p.rot2 ? -si : si);
          turned[c] |= uint32_t(turn) << e;
          const uint32_t at = uint32_t(y * int(sizeof(E)));
          far[e / 2] = e % 2 ? far[e / 2] | at << 16 : at;
        }
      }
    }
  }

  int st = 0;
#pragma unroll 1
  for (int pass = first_pass * step; pass < last; pass += step, hd += step, dst += dst_step) {
    const bool live = store && hd < last;
    cp_async_wait<kRotDepth - 1>();
    if constexpr (FORM == kShifted) __syncwarp();
    P x[CPL][2];
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int j = c * lg + sub;
      x[c][0].zero(), x[c][1].zero();
      if (j < pairs) {
        x[c][0].raw = *reinterpret_cast<const decltype(P::raw)*>(slot_of(st, c, 0));
        x[c][1].raw = *reinterpret_cast<const decltype(P::raw)*>(slot_of(st, c, 1));
      }
    }
    E others[FORM == kShifted ? 2 * V : 1];
    if constexpr (FORM == kShifted) {
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e)
          others[e] = *reinterpret_cast<const E*>(ring + st * PASS + (e % 2 ? far[e / 2] >> 16 : far[e / 2] & 0xffffu));
      }
      __syncwarp();  // every lane has read before the next rows may land here
    }
    fetch(st);
    st = st + 1 == kRotDepth ? 0 : st + 1;
    float f[CPL][2 * V], inv = 1.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      x[c][0].unpack(f[c]);
      x[c][1].unpack(f[c] + V);
    }
    if (w) {  // every lane of the warp takes part in the shuffles, each within its row's group
      float sq = 0.0f;
#pragma unroll
      for (int c = 0; c < CPL; ++c)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) sq = fmaf(f[c][e], f[c][e], sq);
      for (int o = 1; o < lg; o <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      inv = rsqrtf(sq * p.inv_dim + p.eps);
    }
    if (live) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const int j = c * lg + sub;
        if (j < pairs) {
          P y[2] = {x[c][0], x[c][1]};  // values are stored as they came
          if (!is_v) {
            float r[2 * V];
            // a rotation is left out by a branch, not by zeros: 0 * inf would reach the other element
            if constexpr (FORM != kShifted) {
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const int ia = FORM == kNearby ? 2 * e : e, ib = FORM == kNearby ? 2 * e + 1 : V + e;
                const float a = f[c][ia] * inv, b = f[c][ib] * inv;
                r[ia] = a * k1[c][ia];
                r[ib] = b * k1[c][ib];
                if (FORM == kNearby ? (turned[c] >> e & 1) != 0 : turned[c] != 0) {
                  r[ia] = fmaf(b, k2[c][ia], r[ia]);
                  r[ib] = fmaf(a, k2[c][ib], r[ib]);
                }
              }
            } else {
#pragma unroll
              for (int e = 0; e < 2 * V; ++e) {
                r[e] = f[c][e] * inv * k1[c][e];
                if (turned[c] >> e & 1) r[e] = fmaf(Elt<E>::to_f32(others[e]) * inv, k2[c][e], r[e]);
              }
            }
            y[0].pack(r);
            y[1].pack(r + V);
          }
          *reinterpret_cast<decltype(P::raw)*>(dst + at[c][0]) = y[0].raw;
          *reinterpret_cast<decltype(P::raw)*>(dst + at[c][1]) = y[1].raw;
        }
      }
    }
    if constexpr (BITS != 0) {
      if (paged) {
        __syncwarp();
        const E* staged = stage + grp * D;
        const int64_t at = slot + int64_t(hd) * p.P;
        uint8_t* wq = static_cast<uint8_t*>(is_v ? p.v_data : p.k_data) + at * (D * BITS / 8);
        E* sc = static_cast<E*>(is_v ? p.v_scales : p.k_scales) + at * (D / 64);
        E* bi = static_cast<E*>(is_v ? p.v_biases : p.k_biases) + at * (D / 64);
        // head_dim 64 and 128: a lane has 2V neighbours, or 4 where 2V would need more than a warp
        if (V == 1 && D == 128) quantize_part<E, BITS, 4>(staged, wq, sc, bi, sub, live);
        else quantize_part<E, BITS, 2 * V>(staged, wq, sc, bi, sub, live);
        __syncwarp();
      }
    }
  }
  cp_async_wait<0>();
}

template <typename E, int V, int CPL, int BITS>
static const void* rotary_entry(bool trad) {
  return trad ? reinterpret_cast<const void*>(&rotary_kernel<E, V, CPL, BITS, kNearby>)
              : reinterpret_cast<const void*>(&rotary_kernel<E, V, CPL, BITS, kHalves>);
}
template <typename E, int BITS>
static const void* rotary_pick(int vec, bool wide, bool shifted, bool trad) {
  if constexpr (sizeof(E) == 2)
    if (vec == 8) return rotary_entry<E, 8, 1, BITS>(trad);
  if (vec == 4) return shifted ? reinterpret_cast<const void*>(&rotary_kernel<E, 4, 1, BITS, kShifted>) : rotary_entry<E, 4, 1, BITS>(trad);
  if constexpr (BITS == 0) {  // quantized pools have head_dim 64 and 128
    if (wide) return vec == 2 ? rotary_entry<E, 2, 2, BITS>(trad) : rotary_entry<E, 1, 4, BITS>(trad);
  }
  return vec == 2 ? rotary_entry<E, 2, 1, BITS>(trad) : rotary_entry<E, 1, 2, BITS>(trad);
}
template <typename E>
static const void* rotary_bits(int bits, int vec, bool wide, bool shifted, bool trad) {
  return bits == 0   ? rotary_pick<E, 0>(vec, wide, shifted, trad)
         : bits == 4 ? rotary_pick<E, 4>(vec, wide, shifted, trad)
                     : rotary_pick<E, 8>(vec, wide, shifted, trad);
}

const void* rotary_kernel_for(int dtype, int bits, int vec, bool wide, bool shifted, bool traditional) {
  return dtype == 0   ? rotary_bits<float>(bits, vec, wide, shifted, traditional)
         : dtype == 1 ? rotary_bits<__half>(bits, vec, wide, shifted, traditional)
                      : rotary_bits<__nv_bfloat16>(bits, vec, wide, shifted, traditional);
}

// Page dst[i] = page src[i] in every array and layer: a pure copy, bound by
// HBM (every byte read once and written once). Pages are contiguous in each
// array; a block moves one piece of at most kCopyPiece bytes, eight 16-byte
// loads per thread in flight. One block per piece rather than a few that walk
// over many: with a third of the pieces small (the scales and biases of
// quantized pools) the scheduler fills the gaps better, 4.0 GB of pages moved
// in 597 us (6.7 TB/s) against 616 to 700 for 64 down to 8 blocks per SM.
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int unit = blockIdx.x / p.per_pair;  // (layer, pair)
  int piece = blockIdx.x - unit * p.per_pair, a = 0;
  const int layer = unit / p.n, i = unit - layer * p.n;
  const int src = p.src[i], dst = p.dst[i];
  if (src < 0 || src >= p.n_pages || dst < 0 || dst >= p.n_pages) {
    if (p.flags && threadIdx.x == 0) atomicOr(p.flags, kErrBadIndex);
    return;
  }
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
    if (x < n16) v[k] = s[x];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int x = k * kCopyThreads + threadIdx.x;
    if (x < n16) d[x] = v[k];
  }
}

const void* copy_pages_kernel_ptr() { return reinterpret_cast<const void*>(&copy_pages_kernel); }

}  // namespace sd
