// zx_rope_common.h -- rotary positions on the device: the pairs of a head and their rotation.
//
// A pair (x1, x2) of the first rot_dim channels of a head turns by its position's angle:
//   y1 = x1 c - x2 s,   y2 = x2 c + x1 s          (the transpose: s negated)
// with c and s in fp32 from the table row of the position ([rot_dim] = rot_dim / 2 cosines,
// then as many sines).  Pair i is channels (i, i + rot_dim / 2), or (2 i, 2 i + 1) interleaved.
// Both products and their sum are rounded to fp32 (no fused multiply-add), then the result once
// to the tensor's type, so that every path through the library, and a plain evaluation in
// fp32, gives the same bits.
#pragma once

#include "zx_common.h"

namespace zx {

struct RopeTable {
  const float *table;  // [n_pos][rot], 16-byte aligned rows
  int64_t n_pos;
  int32_t rot;  // a multiple of 16
};

// Cosines and sines of pairs 8 p .. 8 p + 8 at table row `row`.
__device__ __forceinline__ void rope_row(const RopeTable &r, int64_t row, int p, float (&c)[8], float (&s)[8]) {
  const float *at = r.table + row * r.rot + 8 * p;
  const float4 c0 = reinterpret_cast<const float4 *>(at)[0], c1 = reinterpret_cast<const float4 *>(at)[1];
  const float4 s0 = reinterpret_cast<const float4 *>(at + r.rot / 2)[0];
  const float4 s1 = reinterpret_cast<const float4 *>(at + r.rot / 2)[1];
  c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
  s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
}

// Turns the 8 pairs of a unit.  a, b: channels 8 p ..+8 and 8 p + rot / 2 ..+8; interleaved,
// channels 16 p ..+8 and 16 p + 8 ..+8.
template <bool INTER>
__device__ __forceinline__ void rope_turn(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8]) {
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x1 = a[2 * i], x2 = a[2 * i + 1], z1 = b[2 * i], z2 = b[2 * i + 1];
      a[2 * i] = x1 * c[i] - x2 * s[i];
      a[2 * i + 1] = x2 * c[i] + x1 * s[i];
      b[2 * i] = z1 * c[4 + i] - z2 * s[4 + i];
      b[2 * i + 1] = z2 * c[4 + i] + z1 * s[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x1 = a[i], x2 = b[i];
      a[i] = x1 * c[i] - x2 * s[i];
      b[i] = x2 * c[i] + x1 * s[i];
    }
  }
}

__device__ __forceinline__ void unpack_bf16x8(uint4 v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = bf_lo(w[i]), f[2 * i + 1] = bf_hi(w[i]);
}
__device__ __forceinline__ uint4 pack_bf16x8(const float (&f)[8]) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// The same on bf16 bits, in place.
template <bool INTER>
__device__ __forceinline__ void rope_turn_bf16(uint4 &a, uint4 &b, const float (&c)[8], const float (&s)[8]) {
  float fa[8], fb[8];
  unpack_bf16x8(a, fa);
  unpack_bf16x8(b, fb);
  rope_turn<INTER>(fa, fb, c, s);
  a = pack_bf16x8(fa);
  b = pack_bf16x8(fb);
}

// The checks of a rotation's arguments that every entry point makes.
inline int rope_check(const char *what, const float *table, int64_t n_pos, int32_t rot, int32_t head_dim) {
  ZX_REQUIRE(table && aligned16(table), "%s: the table must be a 16-byte aligned device pointer", what);
  ZX_REQUIRE(n_pos > 0 && n_pos <= (1LL << 31), "%s: the table must have 1 to 2^31 positions", what);
  ZX_REQUIRE(rot > 0 && rot <= head_dim, "%s: rot_dim %d outside [1, head_dim %d]", what, rot, head_dim);
  if (rot % 16) return fail(ZX_ERR_UNSUPPORTED, "%s: rot_dim %d is not a multiple of 16", what, rot);
  return ZX_OK;
}

}  // namespace zx
