// zx_rope.hip -- rotary positions: the table of cosines and sines, the rotation of query or key
// rows (and its transpose, the gradient), and the FP8 paged append that rotates the keys on the
// way.  All of it is bound by HBM: a row is read and written once, the table's rows come from
// the caches (every head of a row, and every layer of an append, reads the same one).  16,384 rows
// x 32 heads, D = 128, bf16: 43 us, 6.5 TB/s (output and input stay in the memory-side cache);
// 64 rows 3.0 us, most of it the launch; FP8 append, 32 layers x 64 tokens, static scales 5.9 us.
#include <algorithm>

#include "zx_append_common.h"
#include "zx_internal.h"
#include "zx_rope_common.h"

namespace zx {

// ------------------------------------------------------------------ the table

// angle = position * inv_freq in 64 bits: in 32 the angle of position 100,000 is off by up to
// 2^-8 radians.
__global__ void __launch_bounds__(256)
rope_table_kernel(const double *inv_freq, int32_t half, int64_t n_pos, double scale, float *out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n_pos * half) return;
  const int64_t pos = i / half;
  const int32_t j = (int32_t)(i - pos * half);
  double s, c;
  sincos((double)pos * inv_freq[j], &s, &c);
  out[pos * 2 * half + j] = (float)(c * scale);
  out[pos * 2 * half + half + j] = (float)(s * scale);
}

// ------------------------------------------------------------------ the rotation

template <int DT> struct RopeIo;  // 8 values as loaded and stored
template <> struct RopeIo<ZX_BF16> {
  using T = uint16_t;
  static __device__ __forceinline__ void load(const T *p, float (&f)[8]) {
    unpack_bf16x8(*reinterpret_cast<const uint4 *>(p), f);
  }
  static __device__ __forceinline__ void store(T *p, const float (&f)[8]) {
    *reinterpret_cast<uint4 *>(p) = pack_bf16x8(f);
  }
};
template <> struct RopeIo<ZX_F16> {
  using T = uint16_t;
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void load(const T *p, float (&f)[8]) {
    const h8 v = *reinterpret_cast<const h8 *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
  }
  static __device__ __forceinline__ void store(T *p, const float (&f)[8]) {
    h8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (_Float16)f[i];
    *reinterpret_cast<h8 *>(p) = v;
  }
};
template <> struct RopeIo<ZX_F32> {
  using T = float;
  static __device__ __forceinline__ void load(const T *p, float (&f)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ void store(T *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

struct RopeArgs {
  const void *x;
  void *out;
  const int32_t *positions;
  int32_t *err;
  RopeTable r;
  int64_t x_row, x_head, o_row, o_head;  // strides in elements
  uint32_t n_rows;
  int32_t n_heads, head_dim;
  uint32_t units;    // of a head: rot / 16 that turn 8 pairs, then (copy) 8 channels each
  int32_t transpose, copy;  // copy: out is another tensor (the channels past rot are written too)
};

// A thread: one unit of a head.  Neighbouring threads take neighbouring units, then heads, then
// rows: whole cache lines, and the table's row comes from the cache (four heads per thread, so
// that it is read once for them, gained nothing: 4,096 x 32 x 128 bf16 12.6 us either way).
template <int DT, bool INTER> __global__ void __launch_bounds__(256) rope_kernel(RopeArgs a) {
  using Io = RopeIo<DT>;
  using T = typename Io::T;
  const uint32_t per_row = a.units * (uint32_t)a.n_heads;
  const uint32_t at = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = at / per_row;
  if (row >= a.n_rows) return;
  const uint32_t rest = at - row * per_row;
  const uint32_t h = rest / a.units, u = rest - h * a.units;
  const int32_t pos = a.positions[row];
  const T *x = static_cast<const T *>(a.x) + row * a.x_row + h * a.x_head;
  T *out = static_cast<T *>(a.out) + row * a.o_row + h * a.o_head;
  const uint32_t turning = (uint32_t)a.r.rot / 16;
  float f[8], g[8];
  if (u >= turning) {  // 8 channels past rot
    const int c0 = a.r.rot + 8 * (int)(u - turning);
    Io::load(x + c0, f);
    Io::store(out + c0, f);
    return;
  }
  const int ca = INTER ? 16 * u : 8 * u, cb = INTER ? ca + 8 : ca + a.r.rot / 2;
  if (pos < 0 || pos >= a.r.n_pos) {  // no row of the table: as it is
    if (rest == 0 && a.err) atomicOr(a.err, ZX_KERR_POS_RANGE);
    if (a.copy) {
      Io::load(x + ca, f);
      Io::load(x + cb, g);
      Io::store(out + ca, f);
      Io::store(out + cb, g);
    }
    return;
  }
  float c[8], s[8];
  rope_row(a.r, pos, u, c, s);
  Io::load(x + ca, f);
  Io::load(x + cb, g);
  if (a.transpose) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = -s[i];
  }
  rope_turn<INTER>(f, g, c, s);
  Io::store(out + ca, f);
  Io::store(out + cb, g);
}

// ------------------------------------------------------------------ FP8 append with rotation

// Rows x[n_tok][2][H][D] bf16.  Thread t of a block owns unit t % n_unit of rows t / n_unit +
// rpb * k: 16 channels of one (kv, head), as two 16-byte columns that hold whole pairs (K), so a
// unit turns by itself and one scale, or one maximum, per thread suffices.
struct RaGeom {
  int32_t n_unit, rpb;  // n_unit = H * D / 8
  int32_t upd;          // units per (kv, head) = D / 16
  int32_t n_slabs, head_dim;
  int64_t n_tok, row_bytes, x_layer_stride;
};
struct RaUnit {
  int32_t slab, p;  // kv * H + head; its unit in the head
  int32_t ca, cb;   // first channels of the two columns within the head
  bool turns;
};
template <bool INTER> __device__ __forceinline__ RaUnit ra_unit(const RaGeom &g, int rot, int u) {
  RaUnit n;
  n.slab = u / g.upd;
  n.p = u - n.slab * g.upd;
  n.turns = n.slab < g.n_slabs / 2 && n.p < rot / 16;
  const bool half = n.turns && !INTER;
  n.ca = (half ? 8 : 16) * n.p;
  n.cb = n.ca + (half ? rot / 2 : 8);
  return n;
}

// A token's page (-1: none) and position (-1: none), found once per call when there are many.
struct TokPlace {
  int32_t page, pos;
};
__global__ void __launch_bounds__(256)
ra_places_kernel(TokGeom g, int64_t limit, int64_t n_tok, TokPlace *places, int32_t *err) {
  const int64_t t[1] = {(int64_t)blockIdx.x * 256 + threadIdx.x};
  if (t[0] >= n_tok) return;
  int64_t page[1], pos[1];
  int32_t e = 0;
  token_places<1>(g, g.cu_seqlens, g.start_pos, limit, t, n_tok, page, pos, e);
  if (e && err) atomicOr(err, e);
  places[t[0]] = TokPlace{(int32_t)page[0], (int32_t)pos[0]};
}

// The same as the single pass takes it: byte offsets into a layer's pool (-1: none) and positions.
__global__ void __launch_bounds__(256)
ra_offsets_kernel(TokGeom g, int64_t limit, int64_t n_tok, int64_t *tok_off, int32_t *tok_pos, int32_t *err) {
  const int64_t t[1] = {(int64_t)blockIdx.x * 256 + threadIdx.x};
  if (t[0] >= n_tok) return;
  int64_t page[1], pos[1];
  int32_t e = 0;
  token_places<1>(g, g.cu_seqlens, g.start_pos, limit, t, n_tok, page, pos, e);
  if (e && err) atomicOr(err, e);
  tok_off[t[0]] = page[0] < 0 ? -1
                              : page[0] * g.page_bytes +
                                    (int64_t)((uint32_t)pos[0] % (uint32_t)g.page_size) * g.head_dim;
  tok_pos[t[0]] = (int32_t)pos[0];
}

template <bool LOCATE>
__device__ __forceinline__ void ra_find(const TokGeom &tg, const TokStage &stage, int64_t limit, const TokPlace *places,
                                        int64_t row, int64_t n_tok, int64_t &page, int64_t &pos, int32_t &e) {
  if constexpr (LOCATE) {
    const int64_t t[1] = {row};
    int64_t pg[1], ps[1];
    token_places<1>(tg, stage, limit, t, n_tok, pg, ps, e);
    page = pg[0];
    pos = ps[0];
  } else {
    const TokPlace p = row < n_tok ? places[row] : TokPlace{-1, -1};
    page = p.page;
    pos = p.pos;
  }
}
// Both columns of a unit; rows past the last one are zeros.
__device__ __forceinline__ void ra_load(__amdgpu_buffer_rsrc_t rsrc, int off, const RaUnit &n, bool last, uint4 &a, uint4 &b) {
  const q_v4u v = last ? __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + 2 * n.ca, 0, 2 /* nontemporal */)
                       : __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + 2 * n.ca, 0, 0);
  const q_v4u w = last ? __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + 2 * n.cb, 0, 2)
                       : __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + 2 * n.cb, 0, 0);
  a = make_uint4(v.x, v.y, v.z, v.w);
  b = make_uint4(w.x, w.y, w.z, w.w);
}

// Pass 1 (dynamic scales): maxima of |rotated K| and |V| of the tokens that have a position.
template <bool LOCATE, bool INTER>
__global__ void __launch_bounds__(512)
rope_append_amax_kernel(const uint16_t *x, RaGeom g, RopeTable r, TokGeom tg, int64_t limit, const TokPlace *places,
                        uint32_t *part /* [L][gridDim.x][2H] */) {
  const int t = threadIdx.x;
  const int rs = t / g.n_unit;
  const RaUnit n = ra_unit<INTER>(g, r.rot, t - rs * g.n_unit);
  const int layer = blockIdx.y;
  const char *xl = reinterpret_cast<const char *>(x + (int64_t)layer * g.x_layer_stride);
  const int64_t step = (int64_t)gridDim.x * g.rpb;
  uint32_t m = 0;  // two packed 16-bit maxima
  int32_t e = 0;
  __shared__ TokStage stage;
  if constexpr (LOCATE) token_stage(tg, stage);
  for (int64_t r0 = (int64_t)blockIdx.x * g.rpb; r0 < g.n_tok; r0 += step) {
    uint4 a, b;
    int64_t page, pos;
    ra_load(q_rsrc(xl + r0 * g.row_bytes, (g.n_tok - r0) * g.row_bytes),
            (int)(rs * g.row_bytes) + 2 * n.slab * g.head_dim, n, false, a, b);
    ra_find<LOCATE>(tg, stage, limit, places, r0 + rs, g.n_tok, page, pos, e);
    if (n.turns) {
      float c[8], s[8];
      rope_row(r, pos < 0 ? 0 : pos, n.p, c, s);
      rope_turn_bf16<INTER>(a, b, c, s);
    }
    if (pos >= 0) m = absmax_acc(absmax_acc(m, a), b);
  }
  const uint32_t mx = group_max(fold16(m), g.upd);
  __shared__ uint32_t red[512];
  red[t] = mx;
  __syncthreads();
  if (rs == 0 && n.p == 0) {
    uint32_t v = mx;
    for (int k = 1; k < g.rpb; ++k) v = max(v, red[k * g.n_unit + t]);
    part[((int64_t)layer * gridDim.x + blockIdx.x) * g.n_slabs + n.slab] = v << 16;
  }
}

// Pass 2: rotate, encode, scatter (rows from the end of the batch first, where the first
// pass has left the caches).  MODE as kv_quant_rows_kernel's: 0 dynamic scales, 1 static, 2 static and
// saturating.
template <int MODE, bool LOCATE, bool INTER>
__global__ void __launch_bounds__(512)
rope_append_rows_kernel(const uint16_t *x, RaGeom g, RopeTable r, TokGeom tg, int64_t limit, const TokPlace *places,
                        const float *scales, uint8_t *pool, int64_t pool_layer_stride, int32_t *err) {
  const int t = threadIdx.x;
  const int rs = t / g.n_unit;
  const RaUnit n = ra_unit<INTER>(g, r.rot, t - rs * g.n_unit);
  const int layer = blockIdx.y;
  const float sc = scales[(int64_t)layer * g.n_slabs + n.slab];
  const QuantScale q = quant_scale(sc);
  const uint32_t s_sign = (__float_as_uint(sc) >> 24) & 0x80u;
  const int64_t r0 = ((int64_t)gridDim.x - 1 - blockIdx.x) * g.rpb;
  const char *xl = reinterpret_cast<const char *>(x + (int64_t)layer * g.x_layer_stride);
  uint8_t *pl = pool + (int64_t)layer * pool_layer_stride + (int64_t)n.slab * tg.page_size * tg.head_dim;
  uint4 a, b;
  int64_t page, pos;
  ra_load(q_rsrc(xl + r0 * g.row_bytes, (g.n_tok - r0) * g.row_bytes),
          (int)(rs * g.row_bytes) + 2 * n.slab * g.head_dim, n, true, a, b);
  int32_t e = 0;
  __shared__ TokStage stage;
  if constexpr (LOCATE) token_stage(tg, stage);
  ra_find<LOCATE>(tg, stage, limit, places, r0 + rs, g.n_tok, page, pos, e);
  if (LOCATE && e && err && layer == 0 && n.slab == 0 && n.p == 0) atomicOr(err, e);
  if (page < 0) return;
  if (n.turns) {
    float c[8], s[8];
    rope_row(r, pos, n.p, c, s);
    rope_turn_bf16<INTER>(a, b, c, s);
  }
  uint2 ea = quant8(a, q), eb = quant8(b, q);
  if (MODE != 0 && q.nan_fix == 0) {
    ea = static_overflow<MODE>(a, ea, s_sign, err);
    eb = static_overflow<MODE>(b, eb, s_sign, err);
  }
  uint8_t *dst = pl + page * tg.page_bytes + (int64_t)((uint32_t)pos % (uint32_t)tg.page_size) * tg.head_dim;
  typedef unsigned int v2u __attribute__((ext_vector_type(2)));
  const v2u wa = {ea.x, ea.y}, wb = {eb.x, eb.y};
  __builtin_nontemporal_store(wa, reinterpret_cast<v2u *>(dst + n.ca));
  __builtin_nontemporal_store(wb, reinterpret_cast<v2u *>(dst + n.cb));
}

// A thread takes one row: two and four in flight were slower throughout (static scales, 8 heads, D
// = 128, in a graph: 2 layers x 16,000 tokens 40.4 / 41.9 / 44.7 us, 4 x 4,000 22.7 / 24.2 / 25.6),
// and so were 2 and 8 blocks per CU in the first pass (2 x 16,000, both passes: 78 and 72, with 4
// 70 us).
constexpr int RA_BPC = 4;
// Up to this many blocks per CU find the places themselves, without a launch for it before (32 layers
// x 16 tokens 4.5 us against 8.0, x 64 5.9 / 8.7, x 128 8.8 / 9.9; x 256, where too many look for
// the same few, 15.7 / 14.5).
constexpr int64_t RA_LOCATE_BPC = 8;

static int64_t ra_amax_grid_x(int64_t n_tok, int32_t rpb, int32_t n_layers) {
  const int64_t tiles = ceil_div(n_tok, rpb);
  const int64_t want = std::max<int64_t>(1, ceil_div((int64_t)num_cus() * RA_BPC, n_layers));
  return std::max<int64_t>(1, std::min(tiles, want));
}

}  // namespace zx

using namespace zx;

extern "C" int zx_rope_table(const double *inv_freq, int32_t rot_dim, int64_t n_pos, double scale, float *out,
                             zx_stream_t stream) {
  clear_error();
  ZX_REQUIRE(inv_freq, "rope_table: null pointer");
  const int rc = rope_check("rope_table", out, n_pos, rot_dim, rot_dim);
  if (rc) return rc;
  const int64_t blocks = ceil_div(n_pos * (rot_dim / 2), 256);
  if (blocks >= (1LL << 31)) return fail(ZX_ERR_UNSUPPORTED, "rope_table: table too large");
  rope_table_kernel<<<(unsigned)blocks, 256, 0, as_stream(stream)>>>(inv_freq, rot_dim / 2, n_pos, scale, out);
  return check_launch("rope_table");
}

// Whether two of n x heads rows of d elements, `row` and `head` elements apart, share one: is some
// (i, j) != (0, 0), |i| < n, |j| < heads, with |i row + j head| < d?  (128 bits: a stride is anything.)
static bool rope_rows_overlap(int64_t n, int64_t heads, int64_t row, int64_t head, int64_t d) {
  if ((n > 1 && row < d) || (heads > 1 && head < d)) return true;
  if (n == 1 || heads == 1) return false;
  typedef __int128 wide;
  const bool by_head = head <= row;
  const wide small = by_head ? head : row, n_small = by_head ? heads : n, large = by_head ? row : head;
  const int64_t n_large = by_head ? n : heads;
  const wide last = (n_small - 1) * small;  // where the last of the near ones begins
  for (int64_t k = 1; k < n_large && k * large < last + d; ++k) {  // (the usual layouts: no step)
    const wide at = k * large, below = at / small;
    if (at - std::min(below, n_small - 1) * small < d) return true;
    if (below + 1 < n_small && (below + 1) * small - at < d) return true;
  }
  return false;
}

extern "C" int zx_rope(const void *x, int dtype, int64_t n_rows, int32_t n_heads, int32_t head_dim, int64_t x_row_stride,
                       int64_t x_head_stride, const float *table, int64_t n_pos, int32_t rot_dim,
                       const int32_t *positions, int32_t flags, void *out, int64_t out_row_stride,
                       int64_t out_head_stride, int32_t *err, zx_stream_t stream) {
  clear_error();
  ZX_REQUIRE(dtype == ZX_BF16 || dtype == ZX_F16 || dtype == ZX_F32, "rope: unknown dtype %d", dtype);
  ZX_REQUIRE(!(flags & ~(ZX_ROPE_INTERLEAVED | ZX_ROPE_TRANSPOSE)), "rope: unknown flag bits 0x%x", (unsigned)flags);
  ZX_REQUIRE(n_rows >= 0 && n_rows < (1LL << 31) && n_heads > 0 && head_dim > 0, "rope: sizes must be positive");
  if (head_dim % 8) return fail(ZX_ERR_UNSUPPORTED, "rope: head_dim %d is not a multiple of 8", head_dim);
  const int rc = rope_check("rope", table, n_pos, rot_dim, head_dim);
  if (rc) return rc;
  if (n_rows == 0) return ZX_OK;
  ZX_REQUIRE(x && out && positions, "rope: null pointer");
  const int64_t vec = dtype == ZX_F32 ? 4 : 8;
  ZX_REQUIRE(aligned16(x) && aligned16(out) && x_row_stride % vec == 0 && x_head_stride % vec == 0 &&
                 out_row_stride % vec == 0 && out_head_stride % vec == 0,
             "rope: every row of x and out must be 16-byte aligned");
  ZX_REQUIRE(x_row_stride >= 0 && x_head_stride >= 0 && out_row_stride >= 0 && out_head_stride >= 0,
             "rope: negative stride");
  ZX_REQUIRE(x != out || (x_row_stride == out_row_stride && x_head_stride == out_head_stride),
             "rope: in place, x and out must have the same strides");
  RopeArgs a;
  a.x = x;
  a.out = out;
  a.positions = positions;
  a.err = err;
  a.r = RopeTable{table, n_pos, rot_dim};
  a.x_row = x_row_stride;
  a.x_head = x_head_stride;
  a.o_row = out_row_stride;
  a.o_head = out_head_stride;
  a.n_rows = (uint32_t)n_rows;
  a.n_heads = n_heads;
  a.head_dim = head_dim;
  a.copy = x != out;
  a.transpose = (flags & ZX_ROPE_TRANSPOSE) != 0;
  a.units = (uint32_t)(rot_dim / 16 + (a.copy ? (head_dim - rot_dim) / 8 : 0));
  const int64_t threads = n_rows * n_heads * a.units;
  if (threads >= (1LL << 32) - 256) return fail(ZX_ERR_UNSUPPORTED, "rope: too many rows");
  ZX_REQUIRE(!rope_rows_overlap(n_rows, n_heads, out_row_stride, out_head_stride, head_dim),
             "rope: rows of out must not overlap");
  const unsigned blocks = (unsigned)ceil_div(threads, 256);
  const hipStream_t st = as_stream(stream);
  const bool inter = flags & ZX_ROPE_INTERLEAVED;
#define ZX_ROPE_LAUNCH(dt)                               \
  if (inter)                                             \
    rope_kernel<dt, true><<<blocks, 256, 0, st>>>(a);    \
  else                                                   \
    rope_kernel<dt, false><<<blocks, 256, 0, st>>>(a);
  if (dtype == ZX_BF16) {
    ZX_ROPE_LAUNCH(ZX_BF16)
  } else if (dtype == ZX_F16) {
    ZX_ROPE_LAUNCH(ZX_F16)
  } else {
    ZX_ROPE_LAUNCH(ZX_F32)
  }
#undef ZX_ROPE_LAUNCH
  return check_launch("rope");
}

// Rows that a block of the append takes at a time.
static int32_t ra_rows_per_block(int32_t n_heads, int32_t head_dim) {
  const int32_t units = n_heads * head_dim / 8;
  return units >= 256 ? 1 : 256 / units;
}
static bool ra_locates(int32_t n_layers, int64_t n_tok, int32_t n_heads, int32_t head_dim) {
  return ceil_div(n_tok, ra_rows_per_block(n_heads, head_dim)) * n_layers <= RA_LOCATE_BPC * num_cus();
}

// Dynamic scales in one cooperative pass (zx_append_fused.hip)?  By the rule of the append that
// does not rotate, if a share fits the registers.  Whole calls, 8 heads, D = 128, one / two
// passes: 76,000 tokens x 2 layers 228 / 298 us, x 16 1485 / 2276; 37,000 (just under half the
// registers) x 2 172 / 149, x 16 1074 / 1098; 19,000 x 16 1033 / 570.
static bool ra_single_pass(int32_t n_layers, int64_t n_tok, int32_t n_heads, int32_t head_dim, int32_t flags) {
  return !(flags & (ZX_APPEND_STATIC_SCALES | ZX_APPEND_TWO_PASS)) && append_fused_holds(n_tok, head_dim) &&
         ((flags & ZX_APPEND_SINGLE_PASS) || append_fused_preferred(n_tok, head_dim, (int64_t)n_layers * 2 * n_heads));
}
static size_t ra_offsets_bytes(int64_t n_tok) {
  return align256((size_t)n_tok * sizeof(int64_t)) + align256((size_t)n_tok * sizeof(int32_t));
}

extern "C" size_t zx_kv_rope_append_workspace_bytes(int32_t n_layers, int64_t n_tok, int32_t n_heads, int32_t head_dim,
                                                    int32_t flags) {
  if (n_layers <= 0 || n_tok <= 0 || n_heads <= 0 || head_dim < 8) return 0;
  const int64_t gx = std::max<int64_t>(1, ceil_div((int64_t)num_cus() * RA_BPC, n_layers));
  const size_t two = (ra_locates(n_layers, n_tok, n_heads, head_dim) ? 0 : align256((size_t)n_tok * sizeof(TokPlace))) +
                     (flags & ZX_APPEND_STATIC_SCALES ? 0 : align256((size_t)gx * n_layers * 2 * n_heads * sizeof(uint32_t)));
  return ra_single_pass(n_layers, n_tok, n_heads, head_dim, flags)
             ? std::max(two, ra_offsets_bytes(n_tok) + append_fused_workspace_bytes(n_layers, n_heads))
             : two;
}

extern "C" int zx_kv_rope_append(const uint16_t *x, int64_t x_layer_stride, int32_t n_layers, int64_t n_tok,
                                 int32_t n_heads, int32_t head_dim, const float *table, int64_t n_pos, int32_t rot_dim,
                                 const int32_t *cu_seqlens, const int32_t *start_pos, int32_t n_seqs,
                                 const int32_t *block_tables, int32_t max_blocks, int32_t page_size, uint8_t *pool,
                                 int64_t pool_layer_stride, int64_t n_pages, float *scales, int32_t flags, int32_t *err,
                                 void *workspace, size_t workspace_bytes, zx_stream_t stream) {
  clear_error();
  ZX_REQUIRE(!(flags & ~(ZX_APPEND_STATIC_SCALES | ZX_APPEND_SATURATE | ZX_APPEND_TWO_PASS | ZX_APPEND_SINGLE_PASS |
                         ZX_ROPE_INTERLEAVED)),
             "kv_rope_append: unknown flag bits 0x%x", (unsigned)flags);
  ZX_REQUIRE((flags & (ZX_APPEND_TWO_PASS | ZX_APPEND_SINGLE_PASS)) != (ZX_APPEND_TWO_PASS | ZX_APPEND_SINGLE_PASS),
             "kv_rope_append: ZX_APPEND_TWO_PASS and ZX_APPEND_SINGLE_PASS together");
  const bool dynamic = !(flags & ZX_APPEND_STATIC_SCALES);
  ZX_REQUIRE(!(dynamic && (flags & ZX_APPEND_SATURATE)), "kv_rope_append: ZX_APPEND_SATURATE needs static scales");
  ZX_REQUIRE(scales && cu_seqlens && block_tables && pool && (x || n_tok == 0), "kv_rope_append: null pointer");
  ZX_REQUIRE(n_layers > 0 && n_layers <= 65535, "kv_rope_append: n_layers out of range");
  ZX_REQUIRE(n_seqs > 0 && max_blocks > 0 && page_size > 0 && n_pages > 0 && n_heads > 0,
             "kv_rope_append: sizes must be positive");
  ZX_REQUIRE(n_tok >= 0 && n_tok < (1LL << 31), "kv_rope_append: n_tok must be in [0, 2^31)");
  ZX_REQUIRE(n_pages < (1LL << 31), "kv_rope_append: n_pages must be below 2^31");
  if (!(head_dim == 64 || head_dim == 128 || head_dim == 256))
    return fail(ZX_ERR_UNSUPPORTED, "kv_rope_append: head_dim %d not in {64, 128, 256}", head_dim);
  const int64_t row = 2LL * n_heads * head_dim;
  if (row > 8192) return fail(ZX_ERR_UNSUPPORTED, "kv_rope_append: 2*H*D = %lld exceeds 8192", (long long)row);
  int rc = rope_check("kv_rope_append", table, n_pos, rot_dim, head_dim);
  if (rc) return rc;
  ZX_REQUIRE(aligned16(x) && aligned16(pool) &&
                 (n_layers == 1 || (x_layer_stride % 8 == 0 && pool_layer_stride % 16 == 0)),
             "kv_rope_append: x and pool (and every layer of them) must be 16-byte aligned");
  const int64_t page_bytes = row * page_size;
  ZX_REQUIRE(n_layers == 1 || x_layer_stride >= n_tok * row, "kv_rope_append: x layer stride smaller than a layer");
  ZX_REQUIRE(n_layers == 1 || pool_layer_stride >= n_pages * page_bytes,
             "kv_rope_append: pool layer stride smaller than a layer's pages");
  const hipStream_t st = as_stream(stream);
  if (n_tok == 0)  // no token: the scales of an empty batch
    return dynamic ? zx_kv_scales(x, 0, n_layers, 0, n_heads, head_dim, scales, stream) : ZX_OK;
  const size_t need = zx_kv_rope_append_workspace_bytes(n_layers, n_tok, n_heads, head_dim, flags);
  ZX_REQUIRE(aligned16(workspace), "kv_rope_append: workspace must be 16-byte aligned");
  if (need && (!workspace || workspace_bytes < need))
    return fail(ZX_ERR_WORKSPACE, "kv_rope_append: workspace %zu < %zu bytes", workspace_bytes, need);
  RaGeom g;
  g.n_unit = (int32_t)(row / 16);
  g.rpb = ra_rows_per_block(n_heads, head_dim);
  g.upd = head_dim / 16;
  g.n_slabs = 2 * n_heads;
  g.head_dim = head_dim;
  g.n_tok = n_tok;
  g.row_bytes = 2 * row;
  g.x_layer_stride = x_layer_stride;
  const RopeTable r = {table, n_pos, rot_dim};
  const TokGeom tg = {cu_seqlens, start_pos, block_tables, n_seqs, max_blocks, page_size, head_dim, n_pages, page_bytes};
  const int64_t limit = std::min((int64_t)max_blocks * page_size, n_pos);
  const bool locate = ra_locates(n_layers, n_tok, n_heads, head_dim);
  const bool inter = flags & ZX_ROPE_INTERLEAVED;
  if (ra_single_pass(n_layers, n_tok, n_heads, head_dim, flags)) {
    int64_t *tok_off = static_cast<int64_t *>(workspace);
    int32_t *tok_pos = reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + align256((size_t)n_tok * sizeof(int64_t)));
    ra_offsets_kernel<<<(unsigned)ceil_div(n_tok, 256), 256, 0, st>>>(tg, limit, n_tok, tok_off, tok_pos, err);
    if ((rc = check_launch("ra_offsets"))) return rc;
    const AppendRope ar = {table, rot_dim, inter, tok_pos};
    rc = append_fused(x, x_layer_stride, n_layers, n_tok, n_heads, head_dim, tok_off, pool, pool_layer_stride, page_size,
                      scales, err, static_cast<char *>(workspace) + ra_offsets_bytes(n_tok), st, &ar);
    if (rc != ZX_ERR_UNSUPPORTED) return rc;
    clear_error();  // this device cannot run the single-pass kernel: two passes below
  }
  TokPlace *places = static_cast<TokPlace *>(workspace);
  uint32_t *part = reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) +
                                                (locate ? 0 : align256((size_t)n_tok * sizeof(TokPlace))));
  if (!locate) {
    ra_places_kernel<<<(unsigned)ceil_div(n_tok, 256), 256, 0, st>>>(tg, limit, n_tok, places, err);
    if ((rc = check_launch("ra_places"))) return rc;
  }
  const int threads = g.n_unit * g.rpb;
  if (dynamic) {
    const unsigned gx = (unsigned)ra_amax_grid_x(n_tok, g.rpb, n_layers);
    const dim3 grid(gx, n_layers);
#define ZX_RA_AMAX(loc, il) \
  rope_append_amax_kernel<loc, il><<<grid, threads, 0, st>>>(x, g, r, tg, limit, places, part)
    if (locate && inter) ZX_RA_AMAX(true, true);
    else if (locate) ZX_RA_AMAX(true, false);
    else if (inter) ZX_RA_AMAX(false, true);
    else ZX_RA_AMAX(false, false);
#undef ZX_RA_AMAX
    if ((rc = check_launch("rope_append_amax"))) return rc;
    if ((rc = finalize_partials(part, (int32_t)gx, g.n_slabs, n_layers, scales, st))) return rc;
  }
  const dim3 grid((unsigned)ceil_div(n_tok, g.rpb), n_layers);
#define ZX_RA_ROWS2(mode, loc, il)                                                                                     \
  rope_append_rows_kernel<mode, loc, il><<<grid, threads, 0, st>>>(x, g, r, tg, limit, places, scales, pool,           \
                                                                  pool_layer_stride, err)
#define ZX_RA_ROWS(mode)                              \
  if (locate && inter) ZX_RA_ROWS2(mode, true, true); \
  else if (locate) ZX_RA_ROWS2(mode, true, false);    \
  else if (inter) ZX_RA_ROWS2(mode, false, true);     \
  else ZX_RA_ROWS2(mode, false, false);
  if (dynamic) {
    ZX_RA_ROWS(0)
  } else if (flags & ZX_APPEND_SATURATE) {
    ZX_RA_ROWS(2)
  } else {
    ZX_RA_ROWS(1)
  }
#undef ZX_RA_ROWS
#undef ZX_RA_ROWS2
  return check_launch("rope_append_rows");
}
