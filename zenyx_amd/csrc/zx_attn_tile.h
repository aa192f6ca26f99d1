// zx_attn_tile.h -- attention on v_mfma_f32_32x32x16: the types' products, tiles in LDS and the operands
// that are read from them.  For cross attention (zx_cross.hip) and shared pages (zx_shared.hip).
//
// A score tile's lanes hold a column each (32 of them, two lanes with 16 rows of the tile each), and 8
// of a lane's values are one B operand of the next product if that product's other operand takes
// the 16 rows in the order 16 c + 8 a + 4 half + b: it is read transposed from LDS
// (ds_read_b64_tr_b16) in that order.
#pragma once

#include "zx_attn_common.h"

namespace zx {

typedef float cr_f32x16 __attribute__((ext_vector_type(16)));
typedef short cr_i16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 cr_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 cr_f16x2 __attribute__((ext_vector_type(2)));

constexpr int CR_THREADS = 256, CR_WAVES = 4;
constexpr int CR_TILE = 64;  // rows of a tile in LDS
constexpr float CR_NONE = -3.402823466e38f;
constexpr float CR_LAZY = 8.0f;  // a maximum is raised when a score exceeds it by more (log2)

struct CrBf16 {
  static constexpr float BIAS = 0.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
  static __device__ __forceinline__ float lo(uint32_t w) { return bf_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return bf_hi(w); }
  static __device__ __forceinline__ cr_f32x16 mfma(att_u32x4 a, att_u32x4 b, cr_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(att_bf16x8, a), __builtin_bit_cast(att_bf16x8, b), c,
                                                   0, 0, 0);
  }
};
// Weights times 2^BIAS: fp16 loses bits of what is below 2^-14.  (bf16 has fp32's exponents.)
struct CrF16 {
  static constexpr float BIAS = 7.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, cr_f16x2{(_Float16)a, (_Float16)b});
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(cr_f16x2, w)[0]; }
  static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(cr_f16x2, w)[1]; }
  static __device__ __forceinline__ cr_f32x16 mfma(att_u32x4 a, att_u32x4 b, cr_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(cr_f16x8, a), __builtin_bit_cast(cr_f16x8, b), c, 0, 0,
                                                  0);
  }
};

// A tile of R rows of D 16-bit values in LDS: rows 64 bytes apart (mod 256), the 16-byte chunks of
// every 64 bytes permuted by an XOR with two bits of the row.  So both ways of reading touch the 64
// banks evenly: 16 lanes that take the same chunk of 16 rows, and 32 that take 64 bytes of 4 rows (rows
// 32 bytes apart, free of conflicts on 32 banks only, made both take twice the cycles), and a
// lane needs two addresses for either, the rest being constant offsets.
template <int D, int R = CR_TILE> struct CrLds {
  static constexpr int ROW = 2 * D + 64;
  static constexpr int BYTES = R * ROW;
  static constexpr int LOADS = R * D / 8 / CR_THREADS;  // 16 bytes each, per thread
  static constexpr int CHUNKS = D / 8;
};
template <int D> __device__ __forceinline__ uint8_t *cr_at(uint8_t *t, int row, int byte) {
  return t + row * CrLds<D>::ROW + (byte ^ (32 * ((row >> 2) & 1) + 16 * ((row >> 3) & 1)));
}
// Row 32 kt + (lane & 31), channels 16 kc + 8 half ..+8: an operand whose rows (or columns) are the tile's.
template <int D> __device__ __forceinline__ att_u32x4 cr_rows(uint8_t *t, int kt, int kc, int lane) {
  const uint8_t *p = cr_at<D>(t, lane & 31, 32 * (kc & 1) + 16 * (lane >> 5));
  return *reinterpret_cast<const att_u32x4 *>(p + 64 * (kc >> 1) + 32 * kt * CrLds<D>::ROW);
}
// Channel 32 dt + (lane & 31) of rows 16 c + 8 a + 4 half + b (a = 0, 1; b = 0 .. 3): a transposed operand.
template <int D> __device__ __forceinline__ att_u32x4 cr_cols(uint8_t *t, int c, int dt, int lane) {
  const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), byte = 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  const uint8_t *p = cr_at<D>(t, row, byte) + 64 * dt + 16 * c * CrLds<D>::ROW;
  const uint8_t *p8 = cr_at<D>(t, row + 8, byte) + 64 * dt + 16 * c * CrLds<D>::ROW;
  typedef __attribute__((address_space(3))) cr_i16x4 *lds_ptr;
  const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p)));
  const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p8)));
  return att_u32x4{x.x, x.y, y.x, y.y};
}
// A tile that is read by rows alone: 16 lanes that take the same chunk of 16 rows touch the 64 banks evenly.
template <int D> struct CrRowsOnly {
  static constexpr int ROW = 2 * D + 16;
  static __device__ __forceinline__ uint8_t *at(uint8_t *t, int row, int byte) { return t + row * ROW + byte; }
};
// 16 values of a product's column as the two operands of the next product.
template <class T> __device__ __forceinline__ void cr_operands(const float (&x)[16], att_u32x4 (&o)[2]) {
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[c][i] = T::pack(x[8 * c + 2 * i], x[8 * c + 2 * i + 1]);
}

__device__ __forceinline__ float cr_halves_sum(float v) {
  float x, y;
  xrow_pair32(v, x, y);
  return x + y;
}
__device__ __forceinline__ float cr_halves_max(float v) {
  float x, y;
  xrow_pair32(v, x, y);
  return fmaxf(x, y);
}
__device__ __forceinline__ cr_f32x16 cr_zero() {
  cr_f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}
// Row of value i of a product's column.
__device__ __forceinline__ int cr_row(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

}  // namespace zx
