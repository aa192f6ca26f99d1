// zx_attention4.hip -- attention straight from the paged 4-bit pool (zx_kv4_common.h): one query
// token per sequence (decode), and blocks of queries (prefill).
//
//   s_t = sm_scale * q . K_t,   out = sum_t softmax(s)_t V_t,   K, V = code * power of its block
//
// Decode.  Bound by HBM reads of the pages (17/32 byte per element) once contexts are long.  The
// work is dealt as in zx_attention.hip (zx_attn_deal.h).  A wave takes steps of 32 positions (two
// tiles of 16, each inside one page) and computes the transposed problem on
// v_mfma_f32_16x16x32_bf16, so that a query head is a column of every product and its softmax
// state sits in the lanes of that column:
//   * K: a tile's codes are stored in the order of the A operand (lane 16 kg + n: token n, 16
//     bytes of block kg), so the loads are the operand, without a pass through LDS: one
//     conversion per pair gives bf16 with the block's power applied, exactly;
//   * S^T = K Q^T: lane (n, kg) gets the scores of head n with keys 16 T + 4 kg + i;
//   * P^T stays in those registers as the B operand of O^T += V^T P^T, with k = 8 kg + 4 T + i
//     standing for key 16 T + 4 kg + i, as bf16 hi + lo (2^-17 of a weight);
//   * V: bf16 rows in LDS, read back transposed (ds_read_b64_tr_b16).
// Up to 16 query heads of a KV head share a block; the columns without a head cost nothing that
// counts (a step's products take a quarter of the time its bytes take).
#include <algorithm>

#include "zx_attn_deal.h"
#include "zx_internal.h"
#include "zx_kv4_common.h"

namespace zx {

typedef short a4_i16x4 __attribute__((ext_vector_type(4)));
constexpr int A4_STEP = 32;   // positions per wave and step
constexpr int A4_HEADS = 16;  // columns of a product

// What a lane holds of a 16-token tile: CW words of codes, NB power bytes.  D = 128: block kg of
// token n.  D = 64: half (kg & 1) of block kg / 2.  D = 256: blocks kg and kg + 4.
template <int D> struct A4Tile {
  static constexpr int CW = D / 32;
  static constexpr int NB = D == 256 ? 2 : 1;
  uint32_t c[CW];
  uint32_t p[NB];
};
// Channel of the first of the 8 that word w of lane row kg holds.
template <int D> __device__ __forceinline__ int a4_channel(int kg, int w) {
  return D == 64 ? 16 * kg + 8 * w : D == 128 ? 32 * kg + 8 * w : 32 * (kg + 4 * (w / 4)) + 8 * (w % 4);
}
template <int D> __device__ __forceinline__ void a4_load(__amdgpu_buffer_rsrc_t rs, int lane, A4Tile<D> &t) {
  const int n = lane & 15, kg = lane >> 4;
  if constexpr (D == 64) {
    typedef unsigned int v2u __attribute__((ext_vector_type(2)));
    const v2u a = __builtin_amdgcn_raw_buffer_load_b64(rs, (kg >> 1) * 256 + n * 16 + (kg & 1) * 8, 0, 2);
    t.c[0] = a.x, t.c[1] = a.y;
    t.p[0] = __builtin_amdgcn_raw_buffer_load_b8(rs, k4_power_off(D) + (kg >> 1) * 16 + n, 0, 2);
  } else {
#pragma unroll
    for (int i = 0; i < A4Tile<D>::NB; ++i) {
      const att_u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(rs, 1024 * i + 16 * lane, 0, 2);
      t.c[4 * i] = a.x, t.c[4 * i + 1] = a.y, t.c[4 * i + 2] = a.z, t.c[4 * i + 3] = a.w;
      t.p[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, k4_power_off(D) + 64 * i + lane, 0, 2);
    }
  }
}
// Word w as 8 bf16.
template <int D> __device__ __forceinline__ att_u32x4 a4_word(const A4Tile<D> &t, int w) {
  uint32_t a, b, c, d;
  k4_decode8(t.c[w], k4_power(t.p[w / 4]), a, b, c, d);
  return att_u32x4{a, b, c, d};
}

template <int D> struct A4Lds {
  static constexpr int VROW = 2 * D + 32;  // bytes of a token's row of V (D = 128: the rows that a
                                           // transposing read touches lie on distinct banks)
  static constexpr int WAVE = A4_STEP * VROW;
};

__device__ __forceinline__ void a4_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 8 weights as a product's operand: bf16 hi, and what is left of them.
__device__ __forceinline__ void a4_split(const float (&p)[8], att_bf16x8 &hi, att_bf16x8 &lo) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    hi[i] = (__bf16)p[i];
    lo[i] = (__bf16)(p[i] - (float)hi[i]);
  }
}

// V^T of 16 channels from 16 jt on as the A operand: lane (m, kg) gets channel 16 jt + m of keys
// 4 kg ..+4 and 16 + 4 kg ..+4 (rows of VROW bytes at vt).
template <int VROW> __device__ __forceinline__ att_bf16x8 a4_vt(const uint8_t *vt, int jt, int n, int kg) {
  const uint8_t *src = vt + (4 * kg + (n >> 2)) * VROW + 2 * (16 * jt + 4 * (n & 3));
  const a4_i16x4 w0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) a4_i16x4 *)(src));
  const a4_i16x4 w1 =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) a4_i16x4 *)(src + 16 * VROW));
  return __builtin_bit_cast(att_bf16x8, att_u32x4{__builtin_bit_cast(uint2, w0).x, __builtin_bit_cast(uint2, w0).y,
                                                  __builtin_bit_cast(uint2, w1).x, __builtin_bit_cast(uint2, w1).y});
}

// g.group heads per block at most; the last group of a KV head may have fewer.
template <int D>
__global__ void __launch_bounds__(ATT_THREADS, 2)
paged_decode4_kernel(const uint16_t *__restrict__ q, AttnGeom g, const uint8_t *__restrict__ pool,
                     const int32_t *__restrict__ block_tables, const int32_t *__restrict__ seq_lens,
                     float *__restrict__ part, uint16_t *__restrict__ out, int32_t *err, void *table) {
  using Lds = A4Lds<D>;
  constexpr int NC = D / 32;  // products per tile of S^T
  constexpr int NT = D / 16;  // tiles of O^T
  AttnRun run = att_locate(g, seq_lens, AttnTable(table, g.n_seqs), blockIdx.x);
  const int grp = g.n_q_heads / g.n_kv_heads;
  const int per_kv = g.n_group / g.n_kv_heads;  // groups of query heads per KV head
  const int h = run.y / per_kv, first = (run.y - h * per_kv) * g.group;
  const int G = min(g.group, grp - first);
  const int hq0 = h * grp + first;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kg = lane >> 4;
  const int tiles = g.page_size / K4_TOK;
  const int64_t page_bytes = 2LL * g.n_kv_heads * tiles * k4_tile_bytes(D);
  const int64_t head_off = (int64_t)h * tiles * k4_tile_bytes(D);
  const int64_t v_off = (int64_t)g.n_kv_heads * tiles * k4_tile_bytes(D);
  const float qs = g.sm_scale * ATT_LOG2E;
  __shared__ __attribute__((aligned(16))) uint8_t lds[ATT_WAVES][Lds::WAVE];
  __shared__ float sm_m[ATT_WAVES][A4_HEADS], sm_l[ATT_WAVES][A4_HEADS];
  uint8_t *vt = lds[wave];
  int32_t e = 0;
  if (g.whole && run.u == run.u_end) att_zero_rows(g, out, G, hq0, run.b, D);
  while (run.u < run.u_end) {
    const int b = run.b;
    const int32_t len = att_len(g, seq_lens, run);
    const uint32_t b_units = att_units(g, len);
    const uint32_t seg_end = (uint32_t)min(run.u_end - run.b_first, (uint64_t)b_units);
    const bool whole_seq = run.u == run.b_first && seg_end == b_units;
    const uint32_t t_begin = (uint32_t)(run.u - run.b_first) * g.unit;
    const uint32_t t_end = min(att_live_len(g, len), seg_end * g.unit);
    if (t_begin < t_end) {
      // positions past the block table are not attended to, and flagged
      if (threadIdx.x == 0 && (int64_t)len > (int64_t)g.max_blocks * g.page_size) e |= ZX_KERR_POS_RANGE;
      const int32_t *bt = block_tables + (int64_t)b * g.max_blocks;
      // q as the B operand: lane (n, kg) holds head n's channels in the order of K's words
      att_bf16x8 qa[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        att_u32x4 w = {0u, 0u, 0u, 0u};
        if (n < G)
          w = *reinterpret_cast<const att_u32x4 *>(q + ((int64_t)b * g.n_q_heads + hq0 + n) * D + a4_channel<D>(kg, c));
        qa[c] = __builtin_bit_cast(att_bf16x8, w);
      }
      att_f32x4 o[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      float m = -INFINITY, l = 0.0f;  // of head n; l over this lane's keys

      // Branch-free as in the 8-bit kernel: a page id is read for a position clamped into the
      // segment, a tile past the end or on a bad page loads through an empty resource.
      const uint32_t t_last = t_end - 1;
      auto tile_page = [&](uint32_t tp) -> int32_t { return bt[page_of(g, min(tp, t_last))]; };
      auto load_tile = [&](uint32_t tp, int32_t page, A4Tile<D> &k, A4Tile<D> &v, int &rows) {
        const int live = tp < t_end ? (int)min((uint32_t)K4_TOK, t_end - tp) : 0;
        const uint32_t tc = min(tp, t_last);
        const uint32_t in_page = tc - page_of(g, tc) * (uint32_t)g.page_size;
        const bool ok = page >= 0 && page < g.n_pages;
        e |= (live > 0 && !ok) ? ZX_KERR_PAGE_RANGE : 0;
        rows = ok ? live : 0;
        const int nrec = rows ? k4_tile_bytes(D) : 0;
        const uint8_t *src =
            pool + (ok ? (int64_t)page * page_bytes + head_off + (int64_t)(in_page / K4_TOK) * k4_tile_bytes(D) : 0);
        a4_load<D>(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(src), (short)0, nrec, 0x00020000), lane, k);
        a4_load<D>(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(src + (ok ? v_off : 0)), (short)0, nrec,
                                                     0x00020000), lane, v);
      };
      auto compute_step = [&](const A4Tile<D> (&k)[2], const A4Tile<D> (&v)[2], const int (&rows)[2]) {
        // V rows into LDS; tokens past the last one as zeros (what a page holds there may be NaN)
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          A4Tile<D> t = v[T];
          if (rows[T] < K4_TOK) {  // uniform
#pragma unroll
            for (int w = 0; w < A4Tile<D>::CW; ++w) t.c[w] = n < rows[T] ? t.c[w] : 0u;
#pragma unroll
            for (int i = 0; i < A4Tile<D>::NB; ++i) t.p[i] = n < rows[T] ? t.p[i] : 127u;
          }
#pragma unroll
          for (int w = 0; w < A4Tile<D>::CW; ++w)
            *reinterpret_cast<att_u32x4 *>(vt + (16 * T + n) * Lds::VROW + 2 * a4_channel<D>(kg, w)) = a4_word<D>(t, w);
        }
        float s[8];  // of head n with keys 16 T + 4 kg + i, log2 units
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          att_f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < NC; ++c)
            sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(att_bf16x8, a4_word<D>(k[T], c)), qa[c], sc,
                                                         0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[4 * T + i] = 4 * kg + i < rows[T] ? sc[i] * qs : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
        const float m_new = fmaxf(m, xrow_max(mx));
        // the accumulators are rescaled only on the steps where some head's maximum grew
        if (__builtin_amdgcn_ballot_w64(m_new > m)) {
          const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
          m = m_new;
          l *= alpha;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][i] *= alpha;
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = s[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[i] - m);  // (a NaN score stays one)
          l += p[i];
        }
        att_bf16x8 ph, pl;
        a4_split(p, ph, pl);
        a4_wave_sync();
#pragma unroll
        for (int jt = 0; jt < NT; ++jt) {
          const att_bf16x8 av = a4_vt<Lds::VROW>(vt, jt, n, kg);
          o[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, ph, o[jt], 0, 0, 0);
          o[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, pl, o[jt], 0, 0, 0);
        }
        a4_wave_sync();
      };

      // wave w takes steps w, w + 4, ...; loads one step ahead, page ids one more
      constexpr uint32_t stride = ATT_WAVES * A4_STEP;
      uint32_t t0 = t_begin + (uint32_t)wave * A4_STEP;
      A4Tile<D> k0[2], v0[2], k1[2], v1[2];
      int r0[2], r1[2];
      int32_t p0[2], p1[2];
      auto pages_of_step = [&](uint32_t ts, int32_t (&p)[2]) {
        p[0] = tile_page(ts);
        p[1] = tile_page(ts + K4_TOK);
      };
      auto load_step = [&](uint32_t ts, const int32_t (&p)[2], A4Tile<D> (&k)[2], A4Tile<D> (&v)[2], int (&rows)[2]) {
        load_tile(ts, p[0], k[0], v[0], rows[0]);
        load_tile(ts + K4_TOK, p[1], k[1], v[1], rows[1]);
      };
      pages_of_step(t0, p0);
      load_step(t0, p0, k0, v0, r0);
      pages_of_step(t0 + stride, p1);
      while (t0 < t_end) {
        load_step(t0 + stride, p1, k1, v1, r1);
        pages_of_step(t0 + 2 * stride, p0);
        compute_step(k0, v0, r0);
        t0 += stride;
        if (t0 >= t_end) break;
        load_step(t0 + stride, p0, k0, v0, r0);
        pages_of_step(t0 + 2 * stride, p1);
        compute_step(k1, v1, r1);
        t0 += stride;
      }

      // l over the four lane rows, then the block's waves meet in LDS (O in the place of V)
      float x, y;
      xrow_pair32(l, x, y);
      xrow_pair16(x + y, x, y);
      l = x + y;
      static_assert(A4_HEADS * D * 4 <= Lds::WAVE, "a wave's O fits where its V was");
      float *acc_w = reinterpret_cast<float *>(vt);
      if (n < G) {
#pragma unroll
        for (int jt = 0; jt < NT; ++jt) *reinterpret_cast<att_f32x4 *>(acc_w + n * D + 16 * jt + 4 * kg) = o[jt];
        if (kg == 0) {
          sm_m[wave][n] = m;
          sm_l[wave][n] = l;
        }
      }
    }
    __syncthreads();
    const float *const accs[ATT_WAVES] = {reinterpret_cast<const float *>(lds[0]), reinterpret_cast<const float *>(lds[1]),
                                          reinterpret_cast<const float *>(lds[2]), reinterpret_cast<const float *>(lds[3])};
    if (t_begin < t_end) att_store<D, A4_HEADS>(g, sm_m, sm_l, accs, part, out, G, hq0, b, run.x, whole_seq, 1.0f);
    run.u = run.b_first + seg_end;
    run.b_first += b_units;
    ++run.b;
    __syncthreads();
  }
  if (e && err) atomicOr(err, e);
}

}  // namespace zx

using namespace zx;

// Query heads per block: as few groups of at most 16 as there can be, of equal size but the last.
static int32_t a4_groups(int32_t grp) { return (int32_t)ceil_div(grp, A4_HEADS); }

static AttnRuns a4_plan(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_blocks,
                        int32_t page_size) {
  const int64_t groups = (int64_t)n_kv_heads * a4_groups(n_q_heads / n_kv_heads);
  return att_runs(n_seqs, groups, 2LL * num_cus(), ATT_WAVES * A4_STEP, max_blocks, page_size);
}

extern "C" size_t zx_paged_attention4_decode_workspace_bytes(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads,
                                                             int32_t head_dim, int32_t max_blocks, int32_t page_size) {
  if (n_seqs <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads || max_blocks <= 0 || page_size <= 0 ||
      page_size % K4_TOK || !(head_dim == 64 || head_dim == 128 || head_dim == 256))
    return 0;
  return att_workspace_bytes(a4_plan(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size), n_seqs, n_q_heads,
                             head_dim);
}

extern "C" int zx_paged_attention4_decode(const uint16_t *q, int32_t n_q_heads, const uint8_t *pool, int64_t n_pages,
                                          int32_t n_kv_heads, int32_t head_dim, int32_t page_size,
                                          const int32_t *block_tables, int32_t max_blocks, const int32_t *seq_lens,
                                          int32_t n_seqs, float sm_scale, uint16_t *out, int32_t *err, void *workspace,
                                          size_t workspace_bytes, zx_stream_t stream) {
  clear_error();
  int rc = k4_check("paged_attention4_decode", n_pages, n_kv_heads, head_dim, page_size);
  if (rc) return rc;
  ZX_REQUIRE(q && pool && block_tables && seq_lens && out, "paged_attention4_decode: null pointer");
  ZX_REQUIRE(aligned16(q) && aligned16(pool) && aligned16(out),
             "paged_attention4_decode: q, pool and out must be 16-byte aligned");
  ZX_REQUIRE(n_q_heads > 0 && max_blocks > 0 && n_seqs > 0, "paged_attention4_decode: sizes must be positive");
  ZX_REQUIRE(n_q_heads % n_kv_heads == 0, "paged_attention4_decode: n_q_heads must be a multiple of n_kv_heads");
  if (n_seqs > 65535) return fail(ZX_ERR_UNSUPPORTED, "paged_attention4_decode: more than 65535 sequences");
  const size_t need =
      zx_paged_attention4_decode_workspace_bytes(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size);
  if (!workspace || workspace_bytes < need)
    return fail(ZX_ERR_WORKSPACE, "paged_attention4_decode: workspace %zu < %zu bytes", workspace_bytes, need);
  const AttnRuns p = a4_plan(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size);
  AttnGeom g = att_geom(p, n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, n_pages, sm_scale);
  const int32_t grp = n_q_heads / n_kv_heads;
  g.group = (int32_t)ceil_div(grp, a4_groups(grp));
  const int64_t gy = (int64_t)n_kv_heads * a4_groups(grp);
  ZX_REQUIRE(p.n_blk * gy < (1LL << 31), "paged_attention4_decode: too many sequences or heads");
  g.n_group = (int32_t)gy;
  const hipStream_t st = as_stream(stream);
  float *part = static_cast<float *>(workspace);
  void *table = part + n_q_heads * (p.n_run + n_seqs) * (2 + head_dim);
  if ((rc = att_make_table(g, seq_lens, table, st))) return rc;
  const unsigned grid = (unsigned)(p.n_blk * gy);
  switch (head_dim) {
    case 64: paged_decode4_kernel<64><<<grid, ATT_THREADS, 0, st>>>(q, g, pool, block_tables, seq_lens, part, out, err, table); break;
    case 128: paged_decode4_kernel<128><<<grid, ATT_THREADS, 0, st>>>(q, g, pool, block_tables, seq_lens, part, out, err, table); break;
    default: paged_decode4_kernel<256><<<grid, ATT_THREADS, 0, st>>>(q, g, pool, block_tables, seq_lens, part, out, err, table); break;
  }
  if ((rc = check_launch("paged_decode4"))) return rc;
  return att_combine(part, g, nullptr, seq_lens, out, table, st);
}
