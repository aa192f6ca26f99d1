// zx_attn_wave.h -- the attention of one wave to pages, and the end of a tile of its columns, for
// 4-bit pages (zx_attention4.hip) and both kinds of page (zx_shared.hip).
#pragma once

#include "zx_attn_deal.h"
#include "zx_kv4_common.h"

namespace zx {

typedef short aw_i16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 aw_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 aw_f16x2 __attribute__((ext_vector_type(2)));
constexpr int AW_STEP = 32;   // positions per wave and step
constexpr int AW_COLS = 16;  // columns of a product (query heads, or pairs of query row and head)
constexpr int AW_STREAM = 2;  // loads of keys that are read once: nontemporal

// Two words of 16-bit values at a time from codes: what a page format's conversions give.
__device__ __forceinline__ uint32_t aw_bf16_of(uint32_t fp8, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)fp8, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)fp8, 1.0f, false));
}
__device__ __forceinline__ uint32_t aw_f16_of(uint32_t fp8, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)fp8, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)fp8, 1.0f, false));
}

// A page format: what a lane (row kg of 16, token n) holds of a 16-token tile of K or V, and its
// words of 8 channels as 16-bit values.
//
// 4 bits: CW words of codes, NB power bytes.  D = 128: block kg of token n.  D = 64: half (kg & 1)
// of block kg / 2.  D = 256: blocks kg and kg + 4.  Values and weights in bf16.
template <int D> struct Page4 {
  static constexpr int DIM = D, BITS = 4;
  static constexpr int WORDS = D / 32;
  static constexpr int NB = D == 256 ? 2 : 1;
  static constexpr bool F16 = false;     // the type of V and of the weights in the second product
  static constexpr float BIAS = 0.0f;    // weights are carried times 2^BIAS
  struct Tile {
    uint32_t c[WORDS];
    uint32_t p[NB];
  };
  static constexpr int tile_bytes() { return k4_tile_bytes(D); }
  // Bytes of a tile that may be read where `live` of its tokens count.
  static __device__ __forceinline__ int readable(int live) { return live ? k4_tile_bytes(D) : 0; }
  // Channel of the first of the 8 that word w of lane row kg holds.
  static __device__ __forceinline__ int channel(int kg, int w) {
    return D == 64 ? 16 * kg + 8 * w : D == 128 ? 32 * kg + 8 * w : 32 * (kg + 4 * (w / 4)) + 8 * (w % 4);
  }
  template <int POLICY> static __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int lane, Tile &t) {
    const int n = lane & 15, kg = lane >> 4;
    if constexpr (D == 64) {
      typedef unsigned int v2u __attribute__((ext_vector_type(2)));
      const v2u a = __builtin_amdgcn_raw_buffer_load_b64(rs, (kg >> 1) * 256 + n * 16 + (kg & 1) * 8, 0, POLICY);
      t.c[0] = a.x, t.c[1] = a.y;
      t.p[0] = __builtin_amdgcn_raw_buffer_load_b8(rs, k4_power_off(D) + (kg >> 1) * 16 + n, 0, POLICY);
    } else {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const att_u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(rs, 1024 * i + 16 * lane, 0, POLICY);
        t.c[4 * i] = a.x, t.c[4 * i + 1] = a.y, t.c[4 * i + 2] = a.z, t.c[4 * i + 3] = a.w;
        t.p[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, k4_power_off(D) + 64 * i + lane, 0, POLICY);
      }
    }
  }
  static __device__ __forceinline__ att_u32x4 key_word(const Tile &t, int w) {
    uint32_t a, b, c, d;
    k4_decode8(t.c[w], k4_power(t.p[w / 4]), a, b, c, d);
    return att_u32x4{a, b, c, d};
  }
  static __device__ __forceinline__ att_u32x4 value_word(const Tile &t, int w) { return key_word(t, w); }
};

// FP8 (e4m3): D / 16 words of four codes; lane kg holds channels 64 i + 16 kg ..+16 of token n, so
// that a load of 16 bytes per lane takes runs of 64 bytes.  K in bf16 beside the queries; V and
// the weights in fp16 (every e4m3 value is one), the weights times 2^7, as prefill has them.
template <int D> struct Page8 {
  static constexpr int DIM = D, BITS = 8;
  static constexpr int WORDS = D / 32;
  static constexpr bool F16 = true;
  static constexpr float BIAS = 7.0f;
  struct Tile {
    uint32_t c[2 * WORDS];
  };
  static constexpr int tile_bytes() { return 16 * D; }
  static __device__ __forceinline__ int readable(int live) { return live * D; }
  static __device__ __forceinline__ int channel(int kg, int w) { return 64 * (w / 2) + 16 * kg + 8 * (w % 2); }
  template <int POLICY> static __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int lane, Tile &t) {
    const int n = lane & 15, kg = lane >> 4;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const att_u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(rs, n * D + 64 * i + 16 * kg, 0, POLICY);
      t.c[4 * i] = a.x, t.c[4 * i + 1] = a.y, t.c[4 * i + 2] = a.z, t.c[4 * i + 3] = a.w;
    }
  }
  static __device__ __forceinline__ att_u32x4 key_word(const Tile &t, int w) {
    return att_u32x4{aw_bf16_of(t.c[2 * w], false), aw_bf16_of(t.c[2 * w], true), aw_bf16_of(t.c[2 * w + 1], false),
                     aw_bf16_of(t.c[2 * w + 1], true)};
  }
  static __device__ __forceinline__ att_u32x4 value_word(const Tile &t, int w) {
    return att_u32x4{aw_f16_of(t.c[2 * w], false), aw_f16_of(t.c[2 * w], true), aw_f16_of(t.c[2 * w + 1], false),
                     aw_f16_of(t.c[2 * w + 1], true)};
  }
  // Bit 7 of every byte that is a NaN code.
  static __device__ __forceinline__ uint32_t nan_bytes(uint32_t c) {
    return ((c & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  }
};

// The scores' factor sm_scale log2(e) as a positive number: a negative one turns q's signs, 0
// makes q zero (then the running maximum is that of the products, and a product masked with
// -infinity stays that).
struct AttnScale {
  float f;
  uint32_t flip, keep;
  __device__ __forceinline__ explicit AttnScale(float s)
      : f(s == 0.0f ? 1.0f : fabsf(s)), flip(s < 0.0f ? 0x80008000u : 0u), keep(s == 0.0f ? 0u : 0xFFFFFFFFu) {}
  __device__ __forceinline__ bool plain() const { return flip == 0u && keep != 0u; }
  __device__ __forceinline__ void turn(att_bf16x8 &x) const {
    att_u32x4 w = __builtin_bit_cast(att_u32x4, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (w[i] ^ flip) & keep;
    x = __builtin_bit_cast(att_bf16x8, w);
  }
};
// A running maximum before the first key.  Finite, so that exp2(-inf - m) is 0 without a case of
// its own; below every finite score.
constexpr float AW_NONE = -3.402823466e38f;
// A running maximum is raised only when a score exceeds it by more than this (log2 units), so
// weights stay at or below 2^8 and the accumulators are rarely rescaled.  Each lane compares the
// scores it has: a column's maximum over its four lanes is formed on the steps that raise one.
constexpr float AW_LAZY = 8.0f;


// The largest of 8 scores, NaN if one is (then the column's row is NaN whatever its maximum): from
// fmaxf the compiler makes an instruction more for every operand, to quiet signalling NaN.  (Not
// by hand in assembly: no wait would be put between a matrix product and its reader.)
__device__ __forceinline__ float aw_max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
__device__ __forceinline__ float aw_max8(const float (&s)[8]) {
  const float x = aw_max3(s[0], s[1], s[2]);
  return aw_max3(aw_max3(s[3], s[4], s[5]), aw_max3(s[6], s[7], x), x);
}

// The sequence of a row: the last one that begins at it or before.
__device__ __forceinline__ int aw_seq_of(const int32_t *cu_q, int32_t n_seqs, int32_t row) {
  int lo = 0, hi = n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu_q[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// V in LDS: a row of bf16 per token, the 16-byte chunks of tokens 4-7 and 12-15 of a tile swapped
// in pairs.  Rows 8 banks apart (mod 32) put the four that a transposing read touches on
// distinct banks, the swap the eight that a 16-byte store does (without it each store took
// twice its cycles, a third of all the kernels' LDS time).
template <int D> struct AttnLds {
  static constexpr int VROW = 2 * D + 32;
  static constexpr int WAVE = AW_STEP * VROW;
  static constexpr int AROW = D + 4;  // floats of a column of accumulators (eight on distinct banks)
};

// Where word w of lane (n, kg) goes: token 16 T + n.
template <class F> __device__ __forceinline__ uint8_t *aw_vrow(uint8_t *vt, int T, int n, int kg, int w) {
  return vt + (16 * T + n) * AttnLds<F::DIM>::VROW + ((2 * F::channel(kg, w)) ^ (16 * ((n >> 2) & 1)));
}

__device__ __forceinline__ void aw_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 8 weights as a product's operand: fp16, or bf16 hi, and (SPLIT) what is left of them.
template <bool F16, bool SPLIT>
__device__ __forceinline__ void aw_weights(const float (&p)[8], att_bf16x8 &hi, att_bf16x8 &lo) {
  static_assert(!(F16 && SPLIT), "weights are split in bf16 only");
  att_u32x4 h, r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F16) {
      h[i] = __builtin_bit_cast(uint32_t, aw_f16x2{(_Float16)p[2 * i], (_Float16)p[2 * i + 1]});
      continue;
    }
    h[i] = pack_bf16(p[2 * i], p[2 * i + 1]);
    if constexpr (SPLIT) r[i] = pack_bf16(p[2 * i] - bf_lo(h[i]), p[2 * i + 1] - bf_hi(h[i]));
  }
  hi = __builtin_bit_cast(att_bf16x8, h);
  if constexpr (SPLIT) lo = __builtin_bit_cast(att_bf16x8, r);
}

// V^T of 16 channels from 16 jt on as the A operand: lane (m, kg) gets channel 16 jt + m of keys
// 4 kg ..+4 and 16 + 4 kg ..+4 (rows of VROW bytes at vt).
template <int VROW> __device__ __forceinline__ att_bf16x8 aw_vt(const uint8_t *vt, int jt, int n, int kg) {
  const uint8_t *src = vt + (4 * kg + (n >> 2)) * VROW + ((32 * jt + 8 * (n & 3)) ^ (16 * (kg & 1)));
  const aw_i16x4 w0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) aw_i16x4 *)(src));
  const aw_i16x4 w1 =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) aw_i16x4 *)(src + 16 * VROW));
  return __builtin_bit_cast(att_bf16x8, att_u32x4{__builtin_bit_cast(uint2, w0).x, __builtin_bit_cast(uint2, w0).y,
                                                  __builtin_bit_cast(uint2, w1).x, __builtin_bit_cast(uint2, w1).y});
}

// V^T times weights.
template <bool F16> __device__ __forceinline__ att_f32x4 aw_pv(att_bf16x8 v, att_bf16x8 p, att_f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(aw_f16x8, v), __builtin_bit_cast(aw_f16x8, p), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p, c, 0, 0, 0);
}

// Where a KV head's tiles are.
struct AttnPages {
  const uint8_t *pool;
  const int32_t *bt;  // the sequence's block table
  int64_t n_pages, page_bytes, head_off, v_off;
  uint32_t page_size, p_magic;
  int32_t p_shift;
  __device__ __forceinline__ uint32_t page_of(uint32_t t) const {
    return (uint32_t)(((uint64_t)t * p_magic) >> (31 + p_shift));
  }
  // The page of position t (uniform), by the scalar cache: a vector load of it would be waited for
  // together with the loads of K and V before it (shared pages, 128 x 32k positions 187 -> 135 us).
  __device__ __forceinline__ int32_t page_id(uint32_t t) const {
    typedef const __attribute__((address_space(4))) int32_t *scalar;
    return reinterpret_cast<scalar>(reinterpret_cast<uintptr_t>(bt))[page_of(t)];
  }
};

// Tokens below `end` of the tile at t: 0 to 16.  Without a difference that wraps where it is not
// chosen: of `t < end ? min(16, end - t) : 0` the compiler's constraint elimination takes the
// difference for one that never does, concludes that t never reaches end, and may drop a loop's
// exit and everything behind it (it did where prefill's loop saw two strides).
__device__ __forceinline__ uint32_t aw_tile_live(uint32_t end, uint32_t t) {
  return min((uint32_t)K4_TOK, end - min(t, end));
}

// The attention of one wave: CT tiles of 16 columns (a column is a query row and head), its
// steps of 32 keys, their softmax and accumulators.  Everything lives in registers; vt is the
// wave's LDS.  EXACT: weights as bf16 hi + lo (2^-17), otherwise rounded once to F's 16-bit type.
// POLICY: of the loads of K and V.  MASK: columns may end before others (lim); without it all see
// every key of a run.
template <class F, int CT, bool EXACT, int POLICY = AW_STREAM, bool MASK = true> struct AttnWave {
  static constexpr int D = F::DIM;
  using Tile = typename F::Tile;
  static constexpr int NC = D / 32;  // products per tile of S^T
  static constexpr int NT = D / 16;  // tiles of O^T
  using Lds = AttnLds<D>;
  const AttnScale qs;
  uint8_t *const vt;
  const int lane, n, kg;
  att_bf16x8 q[CT][NC];
  uint32_t lim[CT];   // keys below it count for the lane's column
  uint32_t lim_all;   // and for every column
  att_f32x4 o[CT][NT], ol[CT];
  // per column: the running maximum, the product that raises it, the sum over this lane's keys
  // (EXACT; otherwise the sum of the rounded weights is a row of ol, against ones)
  float m[CT], top[CT], l[CT];
  int32_t e = 0;

  __device__ __forceinline__ AttnWave(float scale, uint8_t *vt_)
      : qs(scale), vt(vt_), lane(threadIdx.x & 63), n(lane & 15), kg(lane >> 4) {}

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int t = 0; t < NT; ++t) o[ct][t] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      ol[ct] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      m[ct] = top[ct] = AW_NONE;
      l[ct] = 0.0f;
    }
  }
  // Column 16 ct + n's query as the B operand: lane (n, kg) holds its channels in the order of K's words.
  __device__ __forceinline__ void load_q(int ct, const uint16_t *row, bool live) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      att_u32x4 w = {0u, 0u, 0u, 0u};
      if (live) w = *reinterpret_cast<const att_u32x4 *>(row + F::channel(kg, c));
      q[ct][c] = __builtin_bit_cast(att_bf16x8, w);
    }
  }

  // A weight of 0 times a NaN is one, so on a step that some column does not see to its end the
  // values' NaN blocks go into the products as zeros, and are put into the accumulators of the
  // columns that see them here.  bad: lanes (n, kg) whose block i of token t + n is NaN.
  __device__ __forceinline__ void nan_values(uint64_t bad, int i, uint32_t t) {
    constexpr int GROUPS = D == 64 ? 2 : 4;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const uint32_t seen = (1u << aw_tile_live(lim[ct], t)) - 1u;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        const uint32_t tokens = (uint32_t)(bad >> (D == 64 ? 32 * j : 16 * j)) & 0xFFFFu;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int jt = 2 * ((D == 256 && i ? 4 : 0) + j) + half;
            if (tokens & seen) o[ct][jt][k] = __uint_as_float(0x7FC00000u);
          }
      }
    }
  }

  // The same of FP8 pages, whose NaN codes stand alone: ones in their places make a product that
  // counts, for every column and channel, the NaN values that the column sees.
  __device__ __forceinline__ void nan_codes(uint32_t t0, const Tile (&v)[2]) {
    static_assert(F::BITS == 8 || F::BITS == 4, "");
    if constexpr (F::BITS == 8) {
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int w = 0; w < F::WORDS; ++w) {
          att_u32x4 ones;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bad = F::nan_bytes(v[T].c[2 * w + i / 2]) >> (16 * (i & 1));
            ones[i] = (bad & 0x80u ? 0x3C00u : 0u) | (bad & 0x8000u ? 0x3C000000u : 0u);
          }
          *reinterpret_cast<att_u32x4 *>(aw_vrow<F>(vt, T, n, kg, w)) = ones;
        }
      aw_wave_sync();
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float seen[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) seen[j] = t0 + 16 * (j / 4) + 4 * kg + (j % 4) < lim[ct] ? 1.0f : 0.0f;
        att_bf16x8 p, unused;
        aw_weights<true, false>(seen, p, unused);
#pragma unroll
        for (int jt = 0; jt < NT; ++jt) {
          const att_f32x4 count = aw_pv<true>(aw_vt<Lds::VROW>(vt, jt, n, kg), p, att_f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (count[i] > 0.0f) o[ct][jt][i] = __uint_as_float(0x7FC00000u);
        }
      }
      aw_wave_sync();
    }
  }

  // V rows into LDS; tokens past the last one as zeros (what a page holds there may be NaN; FP8
  // pages are not read there).
  __device__ __forceinline__ void store_v(uint32_t t0, const Tile (&v)[2], const int (&rows)[2]) {
    uint32_t drop = 0;  // FP8: all ones where NaN codes are to go into the products as zeros
    if constexpr (F::BITS == 8) {
      if (MASK && t0 + AW_STEP > lim_all) {  // uniform
        uint32_t any = 0;
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < 2 * F::WORDS; ++i) any |= F::nan_bytes(v[T].c[i]);
        if (__builtin_amdgcn_ballot_w64(any != 0)) {
          nan_codes(t0, v);
          drop = 0xFFFFFFFFu;
        }
      }
    }
#pragma unroll
    for (int T = 0; T < 2; ++T) {
      Tile t = v[T];
      if constexpr (F::BITS == 4) {
        if (rows[T] < K4_TOK) {  // uniform
#pragma unroll
          for (int w = 0; w < F::WORDS; ++w) t.c[w] = n < rows[T] ? t.c[w] : 0u;
#pragma unroll
          for (int i = 0; i < F::NB; ++i) t.p[i] = n < rows[T] ? t.p[i] : 127u;
        }
        if (MASK && t0 + AW_STEP > lim_all) {  // uniform
#pragma unroll
          for (int i = 0; i < F::NB; ++i) {
            const uint64_t bad = __builtin_amdgcn_ballot_w64(t.p[i] == K4_NAN);
            if (bad) {
              nan_values(bad, i, t0 + K4_TOK * T);
              t.p[i] = t.p[i] == K4_NAN ? 127u : t.p[i];
            }
          }
        }
      } else if (drop) {  // uniform
#pragma unroll
        for (int i = 0; i < 2 * F::WORDS; ++i) {
          const uint32_t bad = F::nan_bytes(t.c[i]);  // 0x80 -> 0xFF in each byte
          t.c[i] &= ~((bad - (bad >> 7)) | bad);
        }
      }
#pragma unroll
      for (int w = 0; w < F::WORDS; ++w)
        *reinterpret_cast<att_u32x4 *>(aw_vrow<F>(vt, T, n, kg, w)) = F::value_word(t, w);
    }
  }
  __device__ __forceinline__ void scores(const Tile (&k)[2], float (&s)[CT][8]) {
#pragma unroll
    for (int T = 0; T < 2; ++T) {
      att_f32x4 sc[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) sc[ct] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const att_bf16x8 kw = __builtin_bit_cast(att_bf16x8, F::key_word(k[T], c));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sc[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kw, q[ct][c], sc[ct], 0, 0, 0);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[ct][4 * T + i] = sc[ct][i];
    }
  }
  __device__ __forceinline__ void mask(uint32_t t0, const int (&rows)[2], float (&s)[CT][8]) {
    if (rows[0] < K4_TOK || rows[1] < K4_TOK || (MASK && t0 + AW_STEP > lim_all)) {  // uniform
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = 4 * kg + i;
            if (j >= rows[T] || (MASK && t0 + 16 * T + j >= lim[ct])) s[ct][4 * T + i] = -INFINITY;
          }
    }
  }
  // The running maxima, where a score needs it.
  __device__ __forceinline__ void raise(const float (&s)[CT][8]) {
    float mx[CT];
    bool grew = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      mx[ct] = aw_max8(s[ct]);
      grew |= mx[ct] > top[ct];
    }
    if (__builtin_amdgcn_ballot_w64(grew)) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const float m_new = fmaxf(m[ct], xrow_max(mx[ct]) * qs.f - F::BIAS), alpha = __builtin_amdgcn_exp2f(m[ct] - m_new);
        m[ct] = m_new;
        top[ct] = (m_new + (AW_LAZY + F::BIAS)) / qs.f;
        l[ct] *= alpha;
#pragma unroll
        for (int i = 0; i < 4; ++i) ol[ct][i] *= alpha;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[ct][t][i] *= alpha;
      }
    }
  }
  __device__ __forceinline__ void weights(const float (&s)[CT][8], att_bf16x8 (&ph)[CT], att_bf16x8 (&pl)[CT]) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][i], qs.f, -m[ct]));
      if constexpr (EXACT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) l[ct] += p[i];
      }
      aw_weights<F::F16, EXACT>(p, ph[ct], pl[ct]);
    }
  }
  __device__ __forceinline__ void add_v(const att_bf16x8 (&ph)[CT], const att_bf16x8 (&pl)[CT]) {
    if constexpr (!EXACT) {
      constexpr uint32_t ONE = F::F16 ? 0x3C003C00u : 0x3F803F80u;
      const att_bf16x8 ones = __builtin_bit_cast(att_bf16x8, att_u32x4{ONE, ONE, ONE, ONE});
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) ol[ct] = aw_pv<F::F16>(ones, ph[ct], ol[ct]);
    }
#pragma unroll
    for (int jt = 0; jt < NT; ++jt) {
      const att_bf16x8 av = aw_vt<Lds::VROW>(vt, jt, n, kg);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct][jt] = aw_pv<F::F16>(av, ph[ct], o[ct][jt]);
        if constexpr (EXACT) o[ct][jt] = aw_pv<F::F16>(av, pl[ct], o[ct][jt]);
      }
    }
  }

  // Keys [t0, t_end) in steps of 32, `stride` apart, t0 < t_end.  Branch-free: a page id is read
  // for a position clamped into the range, a tile past the end or on a bad page loads through an
  // empty resource.  Page ids are read a step before the loads that they are for.  At D = 64 with
  // one tile of columns the loads go out a step ahead, into a second set of registers (in a graph,
  // 128 x 100-600, 12 heads 16.8 -> 16.5 us, 16 x 1k-8k, 32/8 heads 20.0 -> 19.5, 64 x 8,000 67.2
  // -> 65.8); with more columns or channels, where the set would cost a wave per SIMD, once the
  // step's codes are converted.
  __device__ __forceinline__ void run(const AttnPages &pg, uint32_t t0, uint32_t t_end, uint32_t stride) {
    constexpr bool AHEAD = D * CT <= 64;
    const uint32_t t_last = t_end - 1;
    struct Step {
      Tile k[2], v[2];
      int rows[2];
    };
    int32_t page[2];
    auto pages_of_step = [&](uint32_t ts) {
      page[0] = pg.page_id(min(ts, t_last));
      page[1] = pg.page_id(min(ts + K4_TOK, t_last));
    };
    auto load_tile = [&](uint32_t tp, int32_t id, Tile &k, Tile &v, int &r) {
      // (readfirstlane: uniform, but taken for a vector operand, and the loads then for a loop over lanes)
      const int live = __builtin_amdgcn_readfirstlane((int)aw_tile_live(t_end, tp));
      const uint32_t tc = min(tp, t_last);
      const uint32_t in_page = tc - pg.page_of(tc) * pg.page_size;
      const bool ok = id >= 0 && id < pg.n_pages;
      e |= (live > 0 && !ok) ? ZX_KERR_PAGE_RANGE : 0;
      r = ok ? live : 0;
      const int nrec = F::readable(r);
      const uint8_t *src =
          pg.pool + (ok ? (int64_t)id * pg.page_bytes + pg.head_off + (int64_t)(in_page / K4_TOK) * F::tile_bytes() : 0);
      F::template load<POLICY>(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(src), (short)0, nrec, 0x00020000), lane, k);
      F::template load<POLICY>(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(src + (ok ? pg.v_off : 0)), (short)0, nrec,
                                                   0x00020000), lane, v);
    };
    auto load_step = [&](uint32_t ts, Step &x) {
      load_tile(ts, page[0], x.k[0], x.v[0], x.rows[0]);
      load_tile(ts + K4_TOK, page[1], x.k[1], x.v[1], x.rows[1]);
    };
    att_bf16x8 ph[CT], pl[CT];
    float s[CT][8];
    Step now;
    pages_of_step(t0);
    load_step(t0, now);
    pages_of_step(t0 + stride);
    if (!qs.plain()) {  // (after the loads, which would otherwise wait for q's)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int c = 0; c < NC; ++c) qs.turn(q[ct][c]);
    }
    if constexpr (AHEAD) {
      auto compute = [&](const Step &x) {
        store_v(t0, x.v, x.rows);
        scores(x.k, s);
        mask(t0, x.rows, s);
        raise(s);
        weights(s, ph, pl);
        aw_wave_sync();
        add_v(ph, pl);
        aw_wave_sync();
      };
      Step next;
      while (t0 < t_end) {
        load_step(t0 + stride, next);
        pages_of_step(t0 + 2 * stride);
        compute(now);
        t0 += stride;
        if (t0 >= t_end) break;
        load_step(t0 + stride, now);
        pages_of_step(t0 + 2 * stride);
        compute(next);
        t0 += stride;
      }
    } else {
      while (t0 < t_end) {
        scores(now.k, s);
        __builtin_amdgcn_sched_barrier(0);
        store_v(t0, now.v, now.rows);
        mask(t0, now.rows, s);
        __builtin_amdgcn_sched_barrier(0);
        t0 += stride;
        load_step(t0, now);
        pages_of_step(t0 + stride);
        raise(s);
        weights(s, ph, pl);
        __builtin_amdgcn_sched_barrier(0);
        aw_wave_sync();
        add_v(ph, pl);
        aw_wave_sync();
      }
    }
  }

  // The sum of column 16 ct + n's weights.
  __device__ __forceinline__ float row_sum(int ct) const {
    if constexpr (!EXACT) return ol[ct][0];
    float x, y;
    xrow_pair32(l[ct], x, y);
    xrow_pair16(x + y, x, y);
    return x + y;
  }
  // Column 16 ct + n's finished row (`row`: its D channels) from the wave's own keys alone.
  __device__ __forceinline__ void store_row(int ct, float sum, uint16_t *row) const {
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int jt = 0; jt < NT; ++jt)
      *reinterpret_cast<uint2 *>(row + 16 * jt + 4 * kg) =
          sum == 0.0f ? make_uint2(0u, 0u)
                      : make_uint2(pack_bf16(o[ct][jt][0] * f, o[ct][jt][1] * f), pack_bf16(o[ct][jt][2] * f, o[ct][jt][3] * f));
  }
  // Tile ct's accumulators into the wave's LDS (in the place of V), [column][channel], and its
  // columns' maxima and sums; the first `live` columns.
  __device__ __forceinline__ void spill(int ct, int live, float *sm_m, float *sm_l) {
    static_assert(AW_COLS * Lds::AROW * 4 <= Lds::WAVE, "a tile of O fits where V was");
    float *acc = reinterpret_cast<float *>(vt);
    const float sum = row_sum(ct);
    if (n >= live) return;
#pragma unroll
    for (int jt = 0; jt < NT; ++jt) *reinterpret_cast<att_f32x4 *>(acc + n * Lds::AROW + 16 * jt + 4 * kg) = o[ct][jt];
    if (kg == 0) {
      sm_m[n] = m[ct];
      sm_l[n] = sum;
    }
  }
};

// The end of a tile of columns: thread t has column t / 16, E channels from (t % 16) E on.  (A
// channel per thread and pass, with its column's maxima, divisions and a 2-byte store each,
// took 13 us per tile: 2 x 857 rows, 32 heads, D = 128, on one key 49 us, 26 so; on 1,024
// keys 77, 54 so.)
template <int D> struct AttnEnd {
  static constexpr int E = D / 16;
  static_assert(AW_COLS * 16 == ATT_THREADS, "a thread per sixteenth of a column");
  float M, sum, acc[E];
  static __device__ __forceinline__ int column() { return threadIdx.x >> 4; }
  static __device__ __forceinline__ int channel() { return (threadIdx.x & 15) * E; }
  // Over the block's four waves: the maximum, the sum and the accumulators.
  __device__ __forceinline__ AttnEnd(const float (&sm_m)[ATT_WAVES][AW_COLS], const float (&sm_l)[ATT_WAVES][AW_COLS],
                                   const uint8_t (&lds)[ATT_WAVES][AttnLds<D>::WAVE]) {
    const int j = column();
    M = sm_m[0][j];
#pragma unroll
    for (int w = 1; w < ATT_WAVES; ++w) M = fmaxf(M, sm_m[w][j]);
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < ATT_WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm_m[w][j] - M);  // (maxima are finite)
      sum += f * sm_l[w][j];
      const att_f32x4 *row =
          reinterpret_cast<const att_f32x4 *>(reinterpret_cast<const float *>(lds[w]) + j * AttnLds<D>::AROW + channel());
#pragma unroll
      for (int i = 0; i < E; ++i) acc[i] += f * row[i / 4][i % 4];
    }
  }
  // The finished row (of D channels at `row`), zeros when no key counted.
  __device__ __forceinline__ void store(uint16_t *row) const {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i)
      w[i] = sum == 0.0f ? 0u : pack_bf16(acc[2 * i] / sum, acc[2 * i + 1] / sum);
    if constexpr (E == 4) {
      *reinterpret_cast<uint2 *>(row + channel()) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < E / 8; ++i)
        reinterpret_cast<uint4 *>(row + channel())[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  // A part of it: maximum, sum, accumulators (8-byte aligned).
  __device__ __forceinline__ void store_part(float *pp) const {
#pragma unroll
    for (int i = 0; i < E / 2; ++i)
      reinterpret_cast<float2 *>(pp + 2 + channel())[i] = make_float2(acc[2 * i], acc[2 * i + 1]);
    if (channel() == 0) *reinterpret_cast<float2 *>(pp) = make_float2(M, sum);
  }
};

}  // namespace zx
