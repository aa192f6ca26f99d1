// zx_kv4.hip -- 4-bit KV pages (zx_kv4_common.h): the paged append, with the rotary positions
// of the keys applied on the way, and the gather back to contiguous bf16.  Both are bound by
// HBM: 2 bytes read and 17/32 written per element, and the other way round.  A block's power
// comes from its own 32 values, so there is no pass for maxima and no scale to keep.  16 prompts of
// 1k-8k tokens, 8 heads, D = 128: append 105 us, 4.6 TB/s, gather 95 us, 5.1 TB/s (a copy of this
// size 4.9); one token each of 64 sequences, one layer: 5.1 us in a graph, most of it the launch.
#include <algorithm>

#include "zx_append_common.h"
#include "zx_internal.h"
#include "zx_kv4_common.h"
#include "zx_rope_common.h"

namespace zx {

struct K4Place {
  int32_t page, pos;  // -1: none
};

__global__ void __launch_bounds__(256)
kv4_places_kernel(TokGeom g, int64_t limit, int64_t n_tok, K4Place *places, int32_t *err) {
  const int64_t t[1] = {(int64_t)blockIdx.x * 256 + threadIdx.x};
  if (t[0] >= n_tok) return;
  int64_t page[1], pos[1];
  int32_t e = 0;
  token_places<1>(g, g.cu_seqlens, g.start_pos, limit, t, n_tok, page, pos, e);
  if (e && err) atomicOr(err, e);
  places[t[0]] = K4Place{(int32_t)page[0], (int32_t)pos[0]};
}

struct K4Append {
  const uint16_t *x;  // [L][n_tok][2][H][D]
  int64_t x_layer_stride, n_tok, row_bytes;
  int32_t n_heads;
  RopeTable r;  // rot 0: no rotation
  TokGeom tg;
  int64_t limit;
  const K4Place *places;
  uint8_t *pool;
  int64_t pool_layer_stride;
  int32_t *err;
  int64_t n_grp;  // groups of 16 tokens x (kv, head), one wave each
};

// One wave: 16 tokens of one (kv, head).  It reads their rows as whole cache lines (lane l: 16
// bytes; 1024 / D tokens per load), lays them out in LDS, and lane 16 g + n then takes block g of
// token n (with D = 64 half the lanes, with D = 256 two blocks each), turns it if it is a key,
// and stores 16 bytes of codes and a power: a full tile of a page goes out as 1 KiB without a gap.
constexpr int K4_WAVES = 4;
template <int D, bool ROPE, bool INTER, bool LOCATE>
__global__ void __launch_bounds__(64 * K4_WAVES) kv4_append_kernel(K4Append a) {
  constexpr int ROW = 2 * D + 16;    // bytes of a token's row in LDS (16 of them on distinct banks)
  constexpr int LPT = D / 8;         // 16-byte loads per token
  constexpr int NL = 16 * LPT / 64;  // loads per lane
  constexpr int BLOCKS = D / 32;
  __shared__ __attribute__((aligned(16))) uint8_t lds[K4_WAVES][16 * ROW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t grp = (int64_t)blockIdx.x * K4_WAVES + wave;
  const bool live = grp < a.n_grp;  // uniform
  const int slabs = 2 * a.n_heads;
  const int64_t tg16 = grp / slabs;
  const int slab = (int)(grp - tg16 * slabs);  // neighbours take neighbouring heads of the same tokens
  const int layer = blockIdx.y;
  const int64_t t0 = tg16 * 16;
  const char *src = reinterpret_cast<const char *>(a.x + (int64_t)layer * a.x_layer_stride) + t0 * a.row_bytes +
                    2LL * slab * D;
  // past the last token the loads return zeros
  const int64_t left = live ? (a.n_tok - t0) * a.row_bytes - 2LL * slab * D : 0;
  const __amdgpu_buffer_rsrc_t rs = q_rsrc(live ? src : reinterpret_cast<const char *>(a.x), left);
  q_v4u v[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int at = i * 64 + lane;
    v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)((at / LPT) * a.row_bytes) + 16 * (at % LPT), 0, 2);
  }
  const int n = lane & 15;
  int64_t page[1], pos[1];
  __shared__ TokStage stage;
  if constexpr (LOCATE) token_stage(a.tg, stage);
  if (!live) return;  // (no barrier follows)
  if constexpr (LOCATE) {
    const int64_t t[1] = {t0 + n};
    int32_t e = 0;
    token_places<1>(a.tg, stage, a.limit, t, a.n_tok, page, pos, e);
    if (e && a.err && layer == 0 && slab == 0 && lane < 16) atomicOr(a.err, e);
  } else {
    const K4Place p = t0 + n < a.n_tok ? a.places[t0 + n] : K4Place{-1, -1};
    page[0] = p.page;
    pos[0] = p.pos;
  }
  uint8_t *rows = lds[wave];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int at = i * 64 + lane;
    *reinterpret_cast<q_v4u *>(rows + (at / LPT) * ROW + 16 * (at % LPT)) = v[i];
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const uint8_t *mine = rows + n * ROW;
  auto chunk = [&](int c) { return *reinterpret_cast<const uint4 *>(mine + 16 * c); };  // channels 8 c ..+8
  const uint32_t in_page = (uint32_t)pos[0] % (uint32_t)a.tg.page_size;
  uint8_t *tile = a.pool + (int64_t)layer * a.pool_layer_stride + page[0] * a.tg.page_bytes +
                  ((int64_t)slab * (a.tg.page_size / K4_TOK) + in_page / K4_TOK) * k4_tile_bytes(D);
  for (int g = lane >> 4; g < BLOCKS; g += 4) {
    uint4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = chunk(4 * g + j);
    if (ROPE && slab < a.n_heads && 32 * g < a.r.rot && page[0] >= 0) {
      const float *row = a.r.table + pos[0] * a.r.rot;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 4 * g + j;
        if (8 * c >= a.r.rot) continue;
        float x[8], y[8];
        unpack_bf16x8(w[j], x);
        if constexpr (INTER) {  // pairs 4 c ..+4
          const float4 cs = *reinterpret_cast<const float4 *>(row + 4 * c);
          const float4 sn = *reinterpret_cast<const float4 *>(row + a.r.rot / 2 + 4 * c);
          const float cc[4] = {cs.x, cs.y, cs.z, cs.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = x[2 * i] * cc[i] - x[2 * i + 1] * ss[i];
            y[2 * i + 1] = x[2 * i + 1] * cc[i] + x[2 * i] * ss[i];
          }
        } else {  // the pairs' other channels are half of the rotated ones away
          const int hc = a.r.rot / 16;
          const bool first = c < hc;
          float z[8], cc[8], ss[8];
          unpack_bf16x8(chunk(first ? c + hc : c - hc), z);
          rope_row(a.r, pos[0], first ? c : c - hc, cc, ss);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = first ? x[i] * cc[i] - z[i] * ss[i] : x[i] * cc[i] + z[i] * ss[i];
        }
        w[j] = pack_bf16x8(y);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = absmax_acc(m, w[j]);
    const uint32_t byte = k4_power_byte(fold16(m));
    const bool bad = byte == K4_NAN;
    const float power = bad ? 1.0f : k4_power(byte);
    uint4 o = make_uint4(k4_encode8(w[0], power), k4_encode8(w[1], power), k4_encode8(w[2], power),
                         k4_encode8(w[3], power));
    if (bad) o = make_uint4(0, 0, 0, 0);
    if (page[0] >= 0) {
      *reinterpret_cast<uint4 *>(tile + g * 256 + (in_page % K4_TOK) * 16) = o;
      tile[k4_power_off(D) + g * 16 + in_page % K4_TOK] = (uint8_t)byte;
    }
  }
}

// Gather: a thread takes 8 codes (4 bytes in, 16 out), a wave 512 / D tokens of one tile, so that
// the page is uniform to a wave and each store writes 1 KiB without a gap.
struct K4Gather {
  int32_t n_heads, page_size, max_blocks, out_len;
  int64_t n_pages;
  uint32_t chunks;  // blocks per (sequence, head, kv)
};
constexpr int K4G_U = 4;  // tokens' steps per block (64 x 2,000 positions: 2 95 us, 4 78, 8 92)
template <int D>
__global__ void __launch_bounds__(256)
kv4_gather_kernel(const uint8_t *__restrict__ pool, K4Gather g, const int32_t *__restrict__ block_tables,
                  const int32_t *__restrict__ seq_lens, uint16_t *k_out, uint16_t *v_out, int32_t *err) {
  constexpr int UPT = D / 8;         // units per token
  constexpr int TPW = 64 / UPT;      // tokens per wave and step
  constexpr int STEP = 256 / UPT;    // tokens per block and step
  const uint32_t row = blockIdx.x / g.chunks, chunk = blockIdx.x - row * g.chunks;
  const int kv = (int)(row & 1);
  const uint32_t bh = row >> 1;
  const uint32_t b = bh / (uint32_t)g.n_heads;
  const int h = (int)(bh - b * (uint32_t)g.n_heads);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t len = seq_lens[b];
  const int32_t *bt = block_tables + (int64_t)b * g.max_blocks;
  const int tiles = g.page_size / K4_TOK;
  const int64_t page_bytes = 2LL * g.n_heads * tiles * k4_tile_bytes(D);
  const int tw = lane / UPT, u = lane % UPT;  // token of the wave, unit (8 channels) of the token
  uint16_t *out = (kv ? v_out : k_out) + (int64_t)bh * g.out_len * D;
  const int64_t t_first = chunk * (int64_t)(K4G_U * STEP) + wave * TPW;
  int32_t page[K4G_U];
#pragma unroll
  for (int k = 0; k < K4G_U; ++k) {
    const uint32_t bi = (uint32_t)(t_first + k * STEP) / (uint32_t)g.page_size;  // (below 2^31 + 2^8)
    page[k] = bt[min(bi, (uint32_t)g.max_blocks - 1)];
  }
  uint32_t c[K4G_U], p[K4G_U];
  int32_t e = 0;
#pragma unroll
  for (int k = 0; k < K4G_U; ++k) {
    const int64_t t = t_first + k * STEP;  // uniform: the wave's first token, in a tile with its others
    const uint32_t bi = (uint32_t)t / (uint32_t)g.page_size;
    c[k] = 0;
    p[k] = 127;
    if (t >= len || t >= g.out_len) continue;
    if (bi >= (uint32_t)g.max_blocks) {
      e |= ZX_KERR_POS_RANGE;
    } else if (page[k] < 0 || page[k] >= g.n_pages) {
      e |= ZX_KERR_PAGE_RANGE;
    } else if (t + tw < len) {
      const int in_page = (int)((uint32_t)t - bi * (uint32_t)g.page_size);
      const uint8_t *tile = pool + page[k] * page_bytes +
                            ((int64_t)(kv * g.n_heads + h) * tiles + in_page / K4_TOK) * k4_tile_bytes(D);
      const int n = in_page % K4_TOK + tw;
      c[k] = *reinterpret_cast<const uint32_t *>(tile + (u / 4) * 256 + n * 16 + 4 * (u % 4));
      p[k] = tile[k4_power_off(D) + (u / 4) * 16 + n];
    }
  }
#pragma unroll
  for (int k = 0; k < K4G_U; ++k) {
    const int64_t t = t_first + k * STEP + tw;
    if (t >= g.out_len) continue;
    uint32_t w0, w1, w2, w3;
    k4_decode8(c[k], k4_power(p[k]), w0, w1, w2, w3);
    const q_v4u o = {w0, w1, w2, w3};
    __builtin_nontemporal_store(o, reinterpret_cast<q_v4u *>(out + t * D + 8 * u));
  }
  if (e && err && lane == 0) atomicOr(err, e);
}

// Up to this many waves per CU find the pages themselves, without a launch for it before (8 heads,
// D = 128, in a graph: 32 layers x 16 tokens 5.2 us against 6.8, x 64 7.6 / 9.0, x 256 23.8 / 26.6;
// at twice as many, 4 layers x 4,000, 39.7 / 40.4: no difference).
constexpr int64_t K4_LOCATE_WPC = 32;

}  // namespace zx

using namespace zx;

static bool kv4_locates(int32_t n_layers, int64_t n_tok, int32_t n_heads) {
  return ceil_div(n_tok, 16) * 2 * n_heads * n_layers <= K4_LOCATE_WPC * num_cus();
}

extern "C" size_t zx_kv4_append_workspace_bytes(int32_t n_layers, int64_t n_tok, int32_t n_heads) {
  if (n_layers <= 0 || n_tok <= 0 || n_heads <= 0 || kv4_locates(n_layers, n_tok, n_heads)) return 0;
  return align256((size_t)n_tok * sizeof(K4Place));
}

template <int D>
static void kv4_append_launch(const K4Append &a, bool locate, bool inter, dim3 grid, hipStream_t st) {
  constexpr int T = 64 * K4_WAVES;
  if (locate) {
    if (!a.r.rot) kv4_append_kernel<D, false, false, true><<<grid, T, 0, st>>>(a);
    else if (inter) kv4_append_kernel<D, true, true, true><<<grid, T, 0, st>>>(a);
    else kv4_append_kernel<D, true, false, true><<<grid, T, 0, st>>>(a);
  } else {
    if (!a.r.rot) kv4_append_kernel<D, false, false, false><<<grid, T, 0, st>>>(a);
    else if (inter) kv4_append_kernel<D, true, true, false><<<grid, T, 0, st>>>(a);
    else kv4_append_kernel<D, true, false, false><<<grid, T, 0, st>>>(a);
  }
}

extern "C" int zx_kv4_append(const uint16_t *x, int64_t x_layer_stride, int32_t n_layers, int64_t n_tok, int32_t n_heads,
                             int32_t head_dim, const float *table, int64_t n_pos, int32_t rot_dim,
                             const int32_t *cu_seqlens, const int32_t *start_pos, int32_t n_seqs,
                             const int32_t *block_tables, int32_t max_blocks, int32_t page_size, uint8_t *pool,
                             int64_t pool_layer_stride, int64_t n_pages, int32_t flags, int32_t *err, void *workspace,
                             size_t workspace_bytes, zx_stream_t stream) {
  clear_error();
  ZX_REQUIRE(!(flags & ~ZX_ROPE_INTERLEAVED), "kv4_append: unknown flag bits 0x%x", (unsigned)flags);
  ZX_REQUIRE(table || !(flags & ZX_ROPE_INTERLEAVED), "kv4_append: ZX_ROPE_INTERLEAVED needs a table");
  ZX_REQUIRE(cu_seqlens && block_tables && pool && (x || n_tok == 0), "kv4_append: null pointer");
  ZX_REQUIRE(n_layers > 0 && n_layers <= 65535, "kv4_append: n_layers out of range");
  ZX_REQUIRE(n_seqs > 0 && max_blocks > 0, "kv4_append: sizes must be positive");
  ZX_REQUIRE(n_tok >= 0 && n_tok < (1LL << 31), "kv4_append: n_tok must be in [0, 2^31)");
  int rc = k4_check("kv4_append", n_pages, n_heads, head_dim, page_size);
  if (rc) return rc;
  if (table && (rc = rope_check("kv4_append", table, n_pos, rot_dim, head_dim))) return rc;
  const int64_t row = 2LL * n_heads * head_dim;
  if (row > (1 << 20)) return fail(ZX_ERR_UNSUPPORTED, "kv4_append: 2*H*D = %lld exceeds 2^20", (long long)row);
  ZX_REQUIRE(aligned16(x) && aligned16(pool) &&
                 (n_layers == 1 || (x_layer_stride % 8 == 0 && pool_layer_stride % 16 == 0)),
             "kv4_append: x and pool (and every layer of them) must be 16-byte aligned");
  const int64_t page_bytes = 2LL * n_heads * (page_size / K4_TOK) * k4_tile_bytes(head_dim);
  ZX_REQUIRE(n_layers == 1 || x_layer_stride >= n_tok * row, "kv4_append: x layer stride smaller than a layer");
  ZX_REQUIRE(n_layers == 1 || pool_layer_stride >= n_pages * page_bytes,
             "kv4_append: pool layer stride smaller than a layer's pages");
  if (n_tok == 0) return ZX_OK;
  const size_t need = zx_kv4_append_workspace_bytes(n_layers, n_tok, n_heads);
  ZX_REQUIRE(aligned16(workspace), "kv4_append: workspace must be 16-byte aligned");
  if (need && (!workspace || workspace_bytes < need))
    return fail(ZX_ERR_WORKSPACE, "kv4_append: workspace %zu < %zu bytes", workspace_bytes, need);
  K4Append a;
  a.x = x;
  a.x_layer_stride = x_layer_stride;
  a.n_tok = n_tok;
  a.row_bytes = 2 * row;
  a.n_heads = n_heads;
  a.r = table ? RopeTable{table, n_pos, rot_dim} : RopeTable{nullptr, 0, 0};
  a.tg = TokGeom{cu_seqlens, start_pos, block_tables, n_seqs, max_blocks, page_size, head_dim, n_pages, page_bytes};
  a.limit = std::min((int64_t)max_blocks * page_size, table ? n_pos : (int64_t)1 << 31);
  a.places = static_cast<const K4Place *>(workspace);
  a.pool = pool;
  a.pool_layer_stride = pool_layer_stride;
  a.err = err;
  a.n_grp = ceil_div(n_tok, 16) * 2 * n_heads;
  const int64_t blocks = ceil_div(a.n_grp, K4_WAVES);
  if (blocks >= (1LL << 31)) return fail(ZX_ERR_UNSUPPORTED, "kv4_append: too many rows");
  const hipStream_t st = as_stream(stream);
  const bool locate = kv4_locates(n_layers, n_tok, n_heads);
  if (!locate) {
    kv4_places_kernel<<<(unsigned)ceil_div(n_tok, 256), 256, 0, st>>>(a.tg, a.limit, n_tok,
                                                                      static_cast<K4Place *>(workspace), err);
    if ((rc = check_launch("kv4_places"))) return rc;
  }
  const dim3 grid((unsigned)blocks, (unsigned)n_layers);
  const bool inter = flags & ZX_ROPE_INTERLEAVED;
  switch (head_dim) {
    case 64: kv4_append_launch<64>(a, locate, inter, grid, st); break;
    case 128: kv4_append_launch<128>(a, locate, inter, grid, st); break;
    default: kv4_append_launch<256>(a, locate, inter, grid, st); break;
  }
  return check_launch("kv4_append");
}

extern "C" int zx_kv4_gather_dequant(const uint8_t *pool, int64_t n_pages, int32_t n_heads, int32_t head_dim,
                                     int32_t page_size, const int32_t *block_tables, int32_t max_blocks,
                                     const int32_t *seq_lens, int32_t n_seqs, int32_t out_len, uint16_t *k_out,
                                     uint16_t *v_out, int32_t *err, zx_stream_t stream) {
  clear_error();
  int rc = k4_check("kv4_gather_dequant", n_pages, n_heads, head_dim, page_size);
  if (rc) return rc;
  ZX_REQUIRE(max_blocks > 0 && n_seqs > 0 && out_len >= 0, "kv4_gather_dequant: sizes must be positive");
  if (out_len == 0) return ZX_OK;
  ZX_REQUIRE(pool && block_tables && seq_lens && k_out && v_out, "kv4_gather_dequant: null pointer");
  ZX_REQUIRE(aligned16(pool) && aligned16(k_out) && aligned16(v_out),
             "kv4_gather_dequant: pool, k_out and v_out must be 16-byte aligned");
  K4Gather g;
  g.n_heads = n_heads;
  g.page_size = page_size;
  g.max_blocks = max_blocks;
  g.out_len = out_len;
  g.n_pages = n_pages;
  g.chunks = (uint32_t)ceil_div(out_len, (int64_t)K4G_U * (2048 / head_dim));
  const int64_t blocks = 2LL * n_seqs * n_heads * g.chunks;
  if (blocks >= (1LL << 31)) return fail(ZX_ERR_UNSUPPORTED, "kv4_gather_dequant: output too large");
  const hipStream_t st = as_stream(stream);
  const unsigned n = (unsigned)blocks;
  switch (head_dim) {
    case 64: kv4_gather_kernel<64><<<n, 256, 0, st>>>(pool, g, block_tables, seq_lens, k_out, v_out, err); break;
    case 128: kv4_gather_kernel<128><<<n, 256, 0, st>>>(pool, g, block_tables, seq_lens, k_out, v_out, err); break;
    default: kv4_gather_kernel<256><<<n, 256, 0, st>>>(pool, g, block_tables, seq_lens, k_out, v_out, err); break;
  }
  return check_launch("kv4_gather");
}
