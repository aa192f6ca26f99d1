// zx_append_common.h -- what the paged appends share: where tokens go, buffer resources, and
// the NaN and overflow codes of static FP8 scales.
#pragma once

#include "zx_common.h"

namespace zx {

typedef unsigned int q_v4u __attribute__((ext_vector_type(4)));
__device__ __forceinline__ __amdgpu_buffer_rsrc_t q_rsrc(const void *base, int64_t bytes) {
  const int n = bytes < 0 ? 0 : (bytes > 0x7FFFFFF0 ? 0x7FFFFFF0 : (int)bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, n, 0x00020000);
}

// 0x80 in each byte of w whose low 7 bits are all set (an e4m3 NaN code), else 0.
__device__ __forceinline__ uint32_t nan_code_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// NaN codes of 8 inputs v under a finite static scale (sign bit s_sign, 0 or 0x80).  The
// code is the NaN code S.1111.111 when the quotient x / s is NaN or rounds beyond the e4m3
// range; its sign is that of the IEEE quotient: the sign of x for a NaN x, else
// sign(x) ^ sign(s).  (div_by_scale's correction step turns an infinite quotient into a
// NaN whose sign is the device's default, so the sign is set here.)  A finite x with a
// NaN code overflowed: MODE 1 flags it, MODE 2 also stores +-448 (S.1111.110).  The
// per-element look runs only when some code is a NaN code.
template <int MODE>
__device__ __forceinline__ uint2 static_overflow(uint4 v, uint2 cd, uint32_t s_sign, int32_t *err) {
  if (!(nan_code_bytes(cd.x) | nan_code_bytes(cd.y))) return cd;
  const uint32_t in[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[2] = {cd.x, cd.y};
  bool hit = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t bits = (in[k >> 1] >> (16 * (k & 1))) & 0xFFFFu;
    const uint32_t mag = bits & 0x7FFFu, x_sign = (bits >> 8) & 0x80u;
    const int sh = 8 * (k & 3);
    const uint32_t code = (c[k >> 2] >> sh) & 0xFFu;
    if ((code & 0x7Fu) == 0x7Fu) {
      const uint32_t sign = mag > 0x7F80u ? x_sign : (x_sign ^ s_sign);
      uint32_t fixed = sign | 0x7Fu;
      if (mag < 0x7F80u) {
        hit = true;
        if (MODE == 2) fixed = sign | 0x7Eu;
      }
      c[k >> 2] = (c[k >> 2] & ~(0xFFu << sh)) | (fixed << sh);
    }
  }
  if (hit && err) atomicOr(err, ZX_KERR_OVERFLOW);
  return make_uint2(c[0], c[1]);
}

// Where tokens go: the page tables of an append.
struct TokGeom {
  const int32_t *cu_seqlens, *start_pos, *block_tables;
  int32_t n_seqs, max_blocks, page_size, head_dim;
  int64_t n_pages, page_bytes;
};

// Places of U tokens: the page of each (-1: none, or a bad one), its position in the sequence
// (-1: in no sequence, negative, or at or beyond `limit` <= max_blocks * page_size); *e collects
// the error bits.  The U searches (last b with cu_seqlens[b] <= t) take their steps together,
// so that a step waits for one load.
// cu, start: g.cu_seqlens and g.start_pos (may be NULL), or copies of them in LDS.
template <int U>
__device__ __forceinline__ void token_places(const TokGeom &g, const int32_t *cu, const int32_t *start, int64_t limit,
                                             const int64_t (&t)[U], int64_t n_tok, int64_t (&page)[U],
                                             int64_t (&pos)[U], int32_t &e) {
  int lo[U], hi[U];
#pragma unroll
  for (int k = 0; k < U; ++k) lo[k] = 0, hi[k] = g.n_seqs - 1;
  for (int left = g.n_seqs - 1; left > 0; left >>= 1) {  // hi - lo <= left
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int mid = (lo[k] + hi[k] + 1) >> 1;
      const bool up = cu[mid] <= t[k];
      if (lo[k] < hi[k]) {
        if (up) lo[k] = mid;
        else hi[k] = mid - 1;
      }
    }
  }
  int32_t c0[U], c1[U], p0[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    c0[k] = cu[lo[k]];
    c1[k] = cu[lo[k] + 1];
    p0[k] = start ? start[lo[k]] : 0;
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    page[k] = pos[k] = -1;
    if (t[k] >= n_tok || t[k] < c0[k] || t[k] >= c1[k]) continue;
    const int64_t p = p0[k] + (t[k] - c0[k]);  // below 2^32
    if (p < 0 || p >= limit) {
      e |= ZX_KERR_POS_RANGE;
      continue;
    }
    pos[k] = p;
    const int64_t id = g.block_tables[(int64_t)lo[k] * g.max_blocks + (uint32_t)p / (uint32_t)g.page_size];
    if (id < 0 || id >= g.n_pages) e |= ZX_KERR_PAGE_RANGE;
    else page[k] = id;
  }
}

// The search's tables in LDS, for up to TOK_STAGED sequences: one load of the whole table instead
// of a chain of loads per token.  Every thread of the block calls token_stage (it has a barrier).
constexpr int TOK_STAGED = 256;
struct TokStage {
  int32_t cu[TOK_STAGED + 1], start[TOK_STAGED];
};
__device__ __forceinline__ void token_stage(const TokGeom &g, TokStage &s) {
  if (g.n_seqs > TOK_STAGED) return;
  for (int i = threadIdx.x; i <= g.n_seqs; i += blockDim.x) {
    s.cu[i] = g.cu_seqlens[i];
    if (i < g.n_seqs) s.start[i] = g.start_pos ? g.start_pos[i] : 0;
  }
  __syncthreads();
}
template <int U>
__device__ __forceinline__ void token_places(const TokGeom &g, const TokStage &s, int64_t limit, const int64_t (&t)[U],
                                             int64_t n_tok, int64_t (&page)[U], int64_t (&pos)[U], int32_t &e) {
  if (g.n_seqs <= TOK_STAGED) token_places<U>(g, s.cu, s.start, limit, t, n_tok, page, pos, e);
  else token_places<U>(g, g.cu_seqlens, g.start_pos, limit, t, n_tok, page, pos, e);
}

// Pool offsets (bytes within one layer of FP8 pages) of U tokens' (page, row) bases, or -1.
template <int U>
__device__ __forceinline__ void token_offsets(const TokGeom &g, const int64_t (&t)[U], int64_t n_tok,
                                              int64_t (&off)[U], int32_t &e) {
  int64_t page[U], pos[U];
  token_places<U>(g, g.cu_seqlens, g.start_pos, (int64_t)g.max_blocks * g.page_size, t, n_tok, page, pos, e);
#pragma unroll
  for (int k = 0; k < U; ++k)
    off[k] = page[k] < 0 ? -1
                         : page[k] * g.page_bytes + (int64_t)((uint32_t)pos[k] % (uint32_t)g.page_size) * g.head_dim;
}


}  // namespace zx
