// zx_kv4_common.h -- the 4-bit KV page format, shared by its append, gather and attention.
//
// A block of 32 channels of one token, K or V, head is held as 32 e2m1 codes (values 0, 1/2, 1,
// 3/2, 2, 3, 4, 6 and their negatives) and one power of two 2^(byte - 127), the smallest that
// brings the block's largest magnitude to 6 or below (at least 2^-125).  The OCP microscaling
// block format with that choice of power: gfx950 converts such codes, power included, to bf16
// in one instruction per pair, exactly.  17/32 byte per element.  A block that holds a NaN, an
// infinity or a magnitude of 1.75 x 2^127 and more (whose code times its power is not finite)
// is stored as NaN: byte 255, codes 0.
//
// Pool layout per layer: [n_pages][2][H][P / 16][tile], a tile holding 16 tokens:
//   codes  [D / 32][16 tokens][16 bytes]   channel 2 i of the block in the low bits of byte i
//   powers [D / 32][16 tokens]             one byte each
// 17 D / 2 bytes.  One 16-byte load per lane then gives a wave a 16-token tile in the order in
// which the matrix cores take it (lane 16 g + n: block g of token n), 1 KiB without a gap.
#pragma once

#include "zx_common.h"

namespace zx {

constexpr int K4_TOK = 16;  // tokens per tile
__host__ __device__ constexpr int k4_tile_bytes(int D) { return 17 * D / 2; }
__host__ __device__ constexpr int k4_power_off(int D) { return 8 * D; }  // of the powers in a tile
constexpr uint32_t K4_NAN = 255;      // power byte of a block that is NaN
constexpr uint32_t K4_TOO_LARGE = 0x7F60;  // bf16 magnitude from which a block is NaN

// Power byte of a block from its largest bf16 magnitude (bits): with the magnitude (1 + m / 128)
// 2^(E - 127) <= 6 x 2^e = 1.5 x 2^(e + 2), e + 127 = E - 2, one more if m > 64.
__device__ __forceinline__ uint32_t k4_power_byte(uint32_t amax) {
  if (amax >= K4_TOO_LARGE) return K4_NAN;
  const int b = (int)((amax + 63u) >> 7) - 2;
  return b < 2 ? 2u : (uint32_t)b;
}
// As an fp32 scale operand of the conversions, which take its exponent; byte 255 (an infinity's)
// makes every value a NaN, zero codes too.
__device__ __forceinline__ float k4_power(uint32_t byte) { return __uint_as_float(byte << 23); }

typedef __bf16 k4_bf2 __attribute__((ext_vector_type(2)));
// 8 bf16 (one 16-byte word) -> 8 codes (nearest, ties to the even code).
__device__ __forceinline__ uint32_t k4_encode8(uint4 v, float power) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(k4_bf2, v.x), power, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(k4_bf2, v.y), power, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(k4_bf2, v.z), power, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(k4_bf2, v.w), power, 3);
  return w;
}
// 8 codes -> 8 bf16 as four words, exact.
__device__ __forceinline__ void k4_decode8(uint32_t c, float power, uint32_t &a, uint32_t &b, uint32_t &d, uint32_t &e) {
  a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 0));
  b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 1));
  d = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 2));
  e = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 3));
}

// The checks of a 4-bit pool's geometry that every entry point makes.
inline int k4_check(const char *what, int64_t n_pages, int32_t n_heads, int32_t head_dim, int32_t page_size) {
  ZX_REQUIRE(n_pages > 0 && n_heads > 0 && page_size > 0, "%s: sizes must be positive", what);
  ZX_REQUIRE(n_pages < (1LL << 31), "%s: n_pages must be below 2^31", what);
  if (!(head_dim == 64 || head_dim == 128 || head_dim == 256))
    return fail(ZX_ERR_UNSUPPORTED, "%s: head_dim %d not in {64, 128, 256}", what, head_dim);
  if (page_size % K4_TOK)
    return fail(ZX_ERR_UNSUPPORTED, "%s: page_size %d is not a multiple of 16", what, page_size);
  return ZX_OK;
}

}  // namespace zx
