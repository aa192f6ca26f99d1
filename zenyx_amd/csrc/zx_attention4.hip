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

// The scores' factor sm_scale log2(e) as a positive number: a negative one turns q's signs, 0
// makes q zero (then the running maximum is that of the products, and a product masked with
// -infinity stays that).
struct A4Scale {
  float f;
  uint32_t flip, keep;
  __device__ __forceinline__ explicit A4Scale(float s)
      : f(s == 0.0f ? 1.0f : fabsf(s)), flip(s < 0.0f ? 0x80008000u : 0u), keep(s == 0.0f ? 0u : 0xFFFFFFFFu) {}
  __device__ __forceinline__ att_bf16x8 operand(att_u32x4 w) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (w[i] ^ flip) & keep;
    return __builtin_bit_cast(att_bf16x8, w);
  }
};
// A running maximum before the first key.  Finite, so that exp2(-inf - m) is 0 without a case of
// its own; below every finite score.
constexpr float A4_NONE = -3.402823466e38f;
// A running maximum is raised only when a score exceeds it by more than this (log2 units), so
// weights stay at or below 2^8 and the accumulators are rarely rescaled.
constexpr float A4_LAZY = 8.0f;

__device__ __forceinline__ float a4_max8(const float (&s)[8]) {
  return fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
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
__global__ void __launch_bounds__(ATT_THREADS, D == 256 ? 2 : 3)
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
  const A4Scale qs(g.sm_scale * ATT_LOG2E);
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
        qa[c] = qs.operand(w);
      }
      att_f32x4 o[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      float m = A4_NONE, l = 0.0f;  // of head n; l over this lane's keys

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
        float s[8];  // q . K of head n with keys 16 T + 4 kg + i
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          att_f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < NC; ++c)
            sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(att_bf16x8, a4_word<D>(k[T], c)), qa[c], sc,
                                                         0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[4 * T + i] = 4 * kg + i < rows[T] ? sc[i] : -INFINITY;
        }
        const float mx = xrow_max(a4_max8(s)) * qs.f;
        if (__builtin_amdgcn_ballot_w64(mx > m + A4_LAZY)) {
          const float m_new = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - m_new);
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
          p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], qs.f, -m));
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

// Blocks of queries.  A column of the products is a (query row, head) of one KV head's group: a
// block takes CT tiles of 16 columns, rows row0 .. of one sequence with all the group's heads,
// and its four waves take every fourth step of 32 keys, each with a running softmax of its own,
// merged at the end.  So no wave waits for another within the loop, K goes from memory to the
// operand without LDS, every conversion serves CT products, and a K/V byte read serves 16 CT
// columns: what a block reads is small, the pages have 4 bits.  Bound by the matrix cores and
// the exponentials together for many rows, by the reads for few.
//   EXACT: weights as bf16 hi + lo (2^-17); otherwise rounded once to bf16, and summed so rounded.
// With few tiles the keys of a tile are shared by up to n_split blocks, whose parts
// prefill4_combine_kernel merges.
struct Prefill4Args {
  const uint16_t *q;
  const int32_t *cu_q, *q_pos0, *bt, *kv_len;
  const uint8_t *pool;
  uint16_t *out;
  float *part;  // [tile][split][16 CT columns][2 + D]
  int32_t *err;
  int64_t n_pages;
  int32_t n_q_heads, n_kv_heads, page_size, max_blocks, n_seqs, causal;
  int32_t group, n_group;     // heads per block, groups of them
  int32_t rows;               // query rows per tile: 16 CT / group
  int32_t n_rt, n_split;      // row tiles per sequence, blocks per tile
  int64_t max_rows;           // n_rt * rows
  uint32_t p_magic;
  int32_t p_shift;
  float sm_log2e;
};

// A block's tile, and which steps of 32 keys are this split's.  All uniform.
struct Prefill4Tile {
  int64_t item;  // tile's number
  int b, h, hq0, G, row0, n_rows, split, parts;
  int64_t q_lo;
  int32_t qpos0;    // position of row row0
  int32_t len;      // keys there are
  uint32_t t_begin, t_end;  // keys of this split
};
__device__ __forceinline__ bool p4_locate(const Prefill4Args &a, uint32_t at, Prefill4Tile &t, int32_t &e) {
  // row tiles slowest and last ones first: under a causal mask they see the most keys
  const uint32_t per_rt = (uint32_t)a.n_group * (uint32_t)a.n_seqs;
  t.split = (int)(at % (uint32_t)a.n_split);
  at /= (uint32_t)a.n_split;
  t.item = at;
  const uint32_t rt_rev = at / per_rt, rem = at - rt_rev * per_rt;
  t.b = (int)(rem / (uint32_t)a.n_group);
  const int y = (int)(rem - (uint32_t)t.b * (uint32_t)a.n_group);
  const int grp = a.n_q_heads / a.n_kv_heads, per_kv = a.n_group / a.n_kv_heads;
  t.h = y / per_kv;
  const int first = (y - t.h * per_kv) * a.group;
  t.G = min(a.group, grp - first);
  t.hq0 = t.h * grp + first;
  const int32_t lo = a.cu_q[t.b], hi = a.cu_q[t.b + 1];
  if (rt_rev == 0 && (int64_t)hi - lo > a.max_rows) e |= ZX_KERR_POS_RANGE;
  const int64_t row0 = ((int64_t)a.n_rt - 1 - rt_rev) * a.rows;
  if (row0 >= (int64_t)hi - lo) return false;
  t.row0 = (int)row0;
  t.n_rows = min(a.rows, hi - lo - t.row0);
  t.q_lo = lo;
  int32_t len = a.kv_len[t.b];
  const int64_t cap = (int64_t)a.max_blocks * a.page_size;  // below 2^31
  if (len > cap) {
    e |= ZX_KERR_POS_RANGE;
    len = (int32_t)cap;
  }
  t.len = max(len, 0);
  const int64_t qpos0 = (int64_t)a.q_pos0[t.b] + t.row0;
  t.qpos0 = (int32_t)min(qpos0, (int64_t)INT32_MAX);
  const int64_t end = a.causal ? min((int64_t)t.len, max((int64_t)0, qpos0 + t.n_rows)) : t.len;
  const int64_t units = ceil_div(end, ATT_WAVES * A4_STEP);
  t.parts = (int)max((int64_t)1, min((int64_t)a.n_split, units / 2));
  if (t.split >= t.parts) return false;
  t.t_begin = (uint32_t)(units * t.split / t.parts) * (ATT_WAVES * A4_STEP);
  t.t_end = (uint32_t)min(end, units * (t.split + 1) / t.parts * (ATT_WAVES * A4_STEP));
  return true;
}

// Tiles of 16 columns a block can hold: what leaves two waves per SIMD.
__host__ __device__ constexpr int a4_most_tiles(int D) { return D == 64 ? 4 : D == 128 ? 3 : 1; }
// Blocks per CU (waves per SIMD), by the registers of the tiles' accumulators and queries.
__host__ __device__ constexpr int a4_per_cu(int D, int CT) {
  return D * CT <= 128 ? 4 : D * CT <= 256 && D < 256 ? 3 : 2;
}

template <int D, int CT, bool EXACT>
__global__ void __launch_bounds__(ATT_THREADS, a4_per_cu(D, CT)) paged_prefill4_kernel(Prefill4Args a) {
  using Lds = A4Lds<D>;
  constexpr int NC = D / 32, NT = D / 16;
  Prefill4Tile tl;
  int32_t e = 0;
  const bool work = p4_locate(a, blockIdx.x, tl, e);
  if (!work) {  // block-uniform
    if (e && a.err && threadIdx.x == 0) atomicOr(a.err, e);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kg = lane >> 4;
  const int tiles = a.page_size / K4_TOK;
  const int64_t page_bytes = 2LL * a.n_kv_heads * tiles * k4_tile_bytes(D);
  const int64_t head_off = (int64_t)tl.h * tiles * k4_tile_bytes(D);
  const int64_t v_off = (int64_t)a.n_kv_heads * tiles * k4_tile_bytes(D);
  const A4Scale qs(a.sm_log2e);
  __shared__ __attribute__((aligned(16))) uint8_t lds[ATT_WAVES][Lds::WAVE];
  __shared__ float sm_m[ATT_WAVES][A4_HEADS], sm_l[ATT_WAVES][A4_HEADS];
  uint8_t *vt = lds[wave];
  const int32_t *bt = a.bt + (int64_t)tl.b * a.max_blocks;

  att_bf16x8 qa[CT][NC];
  uint32_t lim[CT];  // keys below it count for the lane's column
  uint32_t lim_all = 0xFFFFFFFFu;
  const int cols = tl.n_rows * tl.G;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = 16 * ct + n, row = c / tl.G;
    const bool live = c < cols;
    lim[ct] = (uint32_t)tl.len;
    if (a.causal) lim[ct] = (uint32_t)min((int64_t)tl.len, max((int64_t)0, (int64_t)tl.qpos0 + row + 1));
    const uint16_t *src = a.q + ((tl.q_lo + tl.row0 + row) * a.n_q_heads + tl.hq0 + (c - row * tl.G)) * (int64_t)D;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      att_u32x4 w = {0u, 0u, 0u, 0u};
      if (live) w = *reinterpret_cast<const att_u32x4 *>(src + a4_channel<D>(kg, k));
      qa[ct][k] = qs.operand(w);
    }
  }
  // the lowest limit of the tile's rows (row 0's): steps below it need no mask
  lim_all = a.causal ? (uint32_t)min((int64_t)tl.len, max((int64_t)0, (int64_t)tl.qpos0 + 1)) : (uint32_t)tl.len;

  att_f32x4 o[CT][NT], ol[CT];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
    for (int t = 0; t < NT; ++t) o[ct][t] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    ol[ct] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    m[ct] = A4_NONE;
    l[ct] = 0.0f;
  }
  const att_bf16x8 ones = __builtin_bit_cast(att_bf16x8, att_u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});

  const uint32_t t_end = tl.t_end, t_last = t_end ? t_end - 1 : 0;
  auto page_of_pos = [&](uint32_t t) { return (uint32_t)(((uint64_t)t * a.p_magic) >> (31 + a.p_shift)); };
  auto tile_page = [&](uint32_t tp) -> int32_t { return bt[page_of_pos(min(tp, t_last))]; };
  auto load_tile = [&](uint32_t tp, int32_t page, A4Tile<D> &k, A4Tile<D> &v, int &rows) {
    const int live = tp < t_end ? (int)min((uint32_t)K4_TOK, t_end - tp) : 0;
    const uint32_t tc = min(tp, t_last);
    const uint32_t in_page = tc - page_of_pos(tc) * (uint32_t)a.page_size;
    const bool ok = page >= 0 && page < a.n_pages;
    e |= (live > 0 && !ok) ? ZX_KERR_PAGE_RANGE : 0;
    rows = ok ? live : 0;
    const int nrec = rows ? k4_tile_bytes(D) : 0;
    const uint8_t *src =
        a.pool + (ok ? (int64_t)page * page_bytes + head_off + (int64_t)(in_page / K4_TOK) * k4_tile_bytes(D) : 0);
    a4_load<D>(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(src), (short)0, nrec, 0x00020000), lane, k);
    a4_load<D>(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(src + (ok ? v_off : 0)), (short)0, nrec,
                                                 0x00020000), lane, v);
  };
  // V rows into LDS, then S^T of both tiles
  auto scores = [&](uint32_t t0, const A4Tile<D> (&k)[2], const A4Tile<D> (&v)[2], const int (&rows)[2], float (&s)[CT][8]) {
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
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int T = 0; T < 2; ++T) {
      att_f32x4 sc[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) sc[ct] = att_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const att_bf16x8 kw = __builtin_bit_cast(att_bf16x8, a4_word<D>(k[T], c));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          sc[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kw, qa[ct][c], sc[ct], 0, 0, 0);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[ct][4 * T + i] = sc[ct][i];
    }
    if (rows[0] < K4_TOK || rows[1] < K4_TOK || t0 + A4_STEP > lim_all) {  // uniform
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = 4 * kg + i;
            if (j >= rows[T] || t0 + 16 * T + j >= lim[ct]) s[ct][4 * T + i] = -INFINITY;
          }
    }
  };
  // softmax and O^T += V^T P^T
  auto weigh = [&](const float (&s)[CT][8]) {
    float mx[CT];
    bool grew = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      mx[ct] = xrow_max(a4_max8(s[ct])) * qs.f;
      grew = grew || mx[ct] > m[ct] + A4_LAZY;
    }
    if (__builtin_amdgcn_ballot_w64(grew)) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const float m_new = fmaxf(m[ct], mx[ct]), alpha = __builtin_amdgcn_exp2f(m[ct] - m_new);
        m[ct] = m_new;
        l[ct] *= alpha;
#pragma unroll
        for (int i = 0; i < 4; ++i) ol[ct][i] *= alpha;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[ct][t][i] *= alpha;
      }
    }
    att_bf16x8 ph[CT], pl[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][i], qs.f, -m[ct]));
      if constexpr (EXACT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) l[ct] += p[i];
        a4_split(p, ph[ct], pl[ct]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) ph[ct][i] = (__bf16)p[i];
        ol[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, ph[ct], ol[ct], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    a4_wave_sync();
#pragma unroll
    for (int jt = 0; jt < NT; ++jt) {
      const att_bf16x8 av = a4_vt<Lds::VROW>(vt, jt, n, kg);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct][jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, ph[ct], o[ct][jt], 0, 0, 0);
        if constexpr (EXACT) o[ct][jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, pl[ct], o[ct][jt], 0, 0, 0);
      }
    }
    a4_wave_sync();
  };

  constexpr uint32_t stride = ATT_WAVES * A4_STEP;
  uint32_t t0 = tl.t_begin + (uint32_t)wave * A4_STEP;
  if (t0 < t_end) {
    // the next step's loads go out once this one's codes are converted (a second set of
    // registers for them would cost the second wave per SIMD), its page ids one step before
    A4Tile<D> k[2], v[2];
    int rows[2];
    int32_t page[2];
    auto pages_of_step = [&](uint32_t ts) {
      page[0] = tile_page(ts);
      page[1] = tile_page(ts + K4_TOK);
    };
    auto load_step = [&](uint32_t ts) {
      load_tile(ts, page[0], k[0], v[0], rows[0]);
      load_tile(ts + K4_TOK, page[1], k[1], v[1], rows[1]);
    };
    pages_of_step(t0);
    load_step(t0);
    pages_of_step(t0 + stride);
    while (t0 < t_end) {
      float s[CT][8];
      scores(t0, k, v, rows, s);
      __builtin_amdgcn_sched_barrier(0);
      t0 += stride;
      load_step(t0);
      pages_of_step(t0 + stride);
      weigh(s);
    }
  }

  // the waves' columns meet in LDS, one tile of 16 after the other (O in the place of V)
  float *acc_w = reinterpret_cast<float *>(vt);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (EXACT) {
      float x, y;
      xrow_pair32(l[ct], x, y);
      xrow_pair16(x + y, x, y);
      l[ct] = x + y;
    } else {
      l[ct] = ol[ct][0];
    }
#pragma unroll
    for (int jt = 0; jt < NT; ++jt) *reinterpret_cast<att_f32x4 *>(acc_w + n * D + 16 * jt + 4 * kg) = o[ct][jt];
    if (kg == 0) {
      sm_m[wave][n] = m[ct];
      sm_l[wave][n] = l[ct];
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < 16 * D; idx += ATT_THREADS) {
      const int j = idx / D, d = idx % D, c = 16 * ct + j;
      if (c >= cols) break;
      float M = sm_m[0][j];
#pragma unroll
      for (int w = 1; w < ATT_WAVES; ++w) M = fmaxf(M, sm_m[w][j]);
      float acc = 0.0f, ll = 0.0f;
#pragma unroll
      for (int w = 0; w < ATT_WAVES; ++w) {
        const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm_m[w][j] - M);
        acc += f * reinterpret_cast<const float *>(lds[w])[j * D + d];
        ll += f * sm_l[w][j];
      }
      if (tl.parts == 1) {
        const int row = c / tl.G;
        const float v = ll == 0.0f ? 0.0f : acc / ll;
        a.out[((tl.q_lo + tl.row0 + row) * a.n_q_heads + tl.hq0 + (c - row * tl.G)) * (int64_t)D + d] =
            (uint16_t)(pack_bf16(v, 0.0f) & 0xFFFFu);
      } else {
        float *pp = a.part + ((tl.item * a.n_split + tl.split) * (16 * CT) + c) * (int64_t)(2 + D);
        pp[2 + d] = acc;
        if (d == 0) {
          pp[0] = M;
          pp[1] = ll;
        }
      }
    }
    __syncthreads();
  }
  if (e && a.err) atomicOr(a.err, e);
}

// Merges the parts of tiles that were cut: one block of D threads per column of a tile.
template <int D>
__global__ void __launch_bounds__(D) prefill4_combine_kernel(Prefill4Args a, int32_t columns) {
  const uint32_t item = blockIdx.x / (uint32_t)columns;
  const int c = (int)(blockIdx.x - item * (uint32_t)columns);
  Prefill4Tile t;
  int32_t e = 0;
  if (!p4_locate(a, item * (uint32_t)a.n_split, t, e) || t.parts == 1 || c >= t.n_rows * t.G) return;
  const int d = threadIdx.x;
  const float *pp = a.part + (t.item * a.n_split * columns + c) * (int64_t)(2 + D);
  const int64_t step = (int64_t)columns * (2 + D);
  float M = -INFINITY, L = 0.0f, A = 0.0f;
  for (int s = 0; s < t.parts; ++s) M = fmaxf(M, pp[s * step]);
  for (int s = 0; s < t.parts; ++s) {
    const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pp[s * step] - M);
    A += f * pp[s * step + 2 + d];
    L += f * pp[s * step + 1];
  }
  const int row = c / t.G;
  const float v = L == 0.0f ? 0.0f : A / L;
  a.out[((t.q_lo + t.row0 + row) * a.n_q_heads + t.hq0 + (c - row * t.G)) * (int64_t)D + d] =
      (uint16_t)(pack_bf16(v, 0.0f) & 0xFFFFu);
}

}  // namespace zx

using namespace zx;

// Query heads per block: as few groups of at most 16 as there can be, of equal size but the last.
static int32_t a4_groups(int32_t grp) { return (int32_t)ceil_div(grp, A4_HEADS); }

static AttnRuns a4_plan(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_blocks,
                        int32_t page_size) {
  const int64_t groups = (int64_t)n_kv_heads * a4_groups(n_q_heads / n_kv_heads);
  return att_runs(n_seqs, groups, (head_dim == 256 ? 2LL : 3LL) * num_cus(), ATT_WAVES * A4_STEP, max_blocks, page_size);
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

// Column tiles per block, by the columns that a sequence can have at most.
static int a4_column_tiles(int64_t columns, int32_t head_dim) {
  const int most = a4_most_tiles(head_dim);
  return columns <= 16 || most == 1 ? 1 : columns <= 32 ? 2 : most;
}

struct Prefill4Plan {
  int ct;
  int32_t group, n_group, rows;
  int64_t n_rt, items, n_split;
};
static Prefill4Plan p4_plan(int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_blocks,
                            int32_t page_size, int32_t n_seqs, int32_t max_q) {
  Prefill4Plan p;
  const int32_t grp = n_q_heads / n_kv_heads;
  p.group = (int32_t)ceil_div(grp, a4_groups(grp));
  p.n_group = n_kv_heads * a4_groups(grp);
  p.ct = a4_column_tiles((int64_t)max_q * p.group, head_dim);
  p.rows = 16 * p.ct / p.group;
  p.n_rt = ceil_div(max_q, p.rows);
  p.items = p.n_rt * p.n_group * n_seqs;
  // parts of a tile where the tiles do not fill the chip; none shorter than 256 keys
  const int64_t units = ceil_div(std::min((int64_t)max_blocks * page_size, (int64_t)INT32_MAX), ATT_WAVES * A4_STEP);
  const int64_t resident = (int64_t)a4_per_cu(head_dim, p.ct) * num_cus();
  p.n_split = std::max<int64_t>(1, std::min(units / 2, resident / std::max<int64_t>(1, p.items)));
  return p;
}

extern "C" size_t zx_paged_attention4_prefill_workspace_bytes(int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                              int32_t page_size, int32_t max_blocks, int32_t n_seqs,
                                                              int32_t max_q_per_seq) {
  if (n_seqs <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads || max_blocks <= 0 || page_size <= 0 ||
      page_size % K4_TOK || max_q_per_seq <= 0 || !(head_dim == 64 || head_dim == 128 || head_dim == 256))
    return 0;
  const Prefill4Plan p = p4_plan(n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, n_seqs, max_q_per_seq);
  return p.n_split > 1 ? (size_t)p.items * p.n_split * 16 * p.ct * (2 + head_dim) * sizeof(float) : 0;
}

template <int D, int CT>
static int p4_launch(const Prefill4Args &a, bool exact, unsigned grid, unsigned items, hipStream_t st) {
  if (CT == 1 || exact)  // (bound by the reads with one tile of columns: the second product is free)
    paged_prefill4_kernel<D, CT, true><<<grid, ATT_THREADS, 0, st>>>(a);
  else if constexpr (CT > 1)
    paged_prefill4_kernel<D, CT, false><<<grid, ATT_THREADS, 0, st>>>(a);
  const int rc = check_launch("paged_prefill4");
  if (rc || a.n_split == 1) return rc;
  prefill4_combine_kernel<D><<<items * 16 * CT, D, 0, st>>>(a, 16 * CT);
  return check_launch("prefill4_combine");
}

extern "C" int zx_paged_attention4_prefill(const uint16_t *q, int64_t n_q, const int32_t *cu_q, const int32_t *q_pos0,
                                           int32_t n_q_heads, const uint8_t *pool, int64_t n_pages, int32_t n_kv_heads,
                                           int32_t head_dim, int32_t page_size, const int32_t *block_tables,
                                           int32_t max_blocks, const int32_t *kv_len, int32_t n_seqs,
                                           int32_t max_q_per_seq, int32_t causal, float sm_scale, int32_t flags,
                                           uint16_t *out, int32_t *err, void *workspace, size_t workspace_bytes,
                                           zx_stream_t stream) {
  clear_error();
  ZX_REQUIRE(!(flags & ~ZX_PREFILL_EXACT_P), "paged_attention4_prefill: unknown flag bits 0x%x", (unsigned)flags);
  int rc = k4_check("paged_attention4_prefill", n_pages, n_kv_heads, head_dim, page_size);
  if (rc) return rc;
  ZX_REQUIRE(n_q >= 0 && max_q_per_seq >= 0 && n_q_heads > 0 && max_blocks > 0 && n_seqs > 0,
             "paged_attention4_prefill: sizes must be positive");
  ZX_REQUIRE(n_q_heads % n_kv_heads == 0, "paged_attention4_prefill: n_q_heads must be a multiple of n_kv_heads");
  ZX_REQUIRE((int64_t)max_blocks * page_size < (1LL << 31),
             "paged_attention4_prefill: block tables of 2^31 positions and more");
  if (n_q == 0 || max_q_per_seq == 0) return ZX_OK;
  ZX_REQUIRE(q && cu_q && q_pos0 && pool && block_tables && kv_len && out, "paged_attention4_prefill: null pointer");
  ZX_REQUIRE(aligned16(q) && aligned16(pool) && aligned16(out),
             "paged_attention4_prefill: q, pool and out must be 16-byte aligned");
  if (max_q_per_seq > n_q) max_q_per_seq = (int32_t)n_q;
  const Prefill4Plan p = p4_plan(n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, n_seqs, max_q_per_seq);
  if (p.items * p.n_split * 16 * p.ct >= (1LL << 31))
    return fail(ZX_ERR_UNSUPPORTED, "paged_attention4_prefill: too many rows");
  Prefill4Args a;
  a.q = q;
  a.cu_q = cu_q;
  a.q_pos0 = q_pos0;
  a.bt = block_tables;
  a.kv_len = kv_len;
  a.pool = pool;
  a.out = out;
  a.part = static_cast<float *>(workspace);
  a.err = err;
  a.n_pages = n_pages;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.page_size = page_size;
  a.max_blocks = max_blocks;
  a.n_seqs = n_seqs;
  a.causal = causal ? 1 : 0;
  a.group = p.group;
  a.n_group = p.n_group;
  a.rows = p.rows;
  a.n_rt = (int32_t)p.n_rt;
  a.max_rows = p.n_rt * p.rows;
  a.sm_log2e = sm_scale * ATT_LOG2E;
  const size_t need = zx_paged_attention4_prefill_workspace_bytes(n_q_heads, n_kv_heads, head_dim, page_size, max_blocks,
                                                                  n_seqs, max_q_per_seq);
  ZX_REQUIRE(!workspace || aligned16(workspace), "paged_attention4_prefill: workspace must be 16-byte aligned");
  a.n_split = need && workspace && workspace_bytes >= need ? (int32_t)p.n_split : 1;
  {
    int sh = 0;
    while ((1LL << sh) < page_size) ++sh;
    a.p_shift = sh;
    a.p_magic = (uint32_t)(((1ULL << (31 + sh)) + (uint64_t)page_size - 1) / (uint64_t)page_size);
  }
  const unsigned items = (unsigned)p.items, grid = items * (unsigned)a.n_split;
  const hipStream_t st = as_stream(stream);
  const bool exact = flags & ZX_PREFILL_EXACT_P;
  constexpr int M64 = a4_most_tiles(64), M128 = a4_most_tiles(128);
  switch (head_dim) {
    case 64:
      return p.ct == 1   ? p4_launch<64, 1>(a, exact, grid, items, st)
             : p.ct == 2 ? p4_launch<64, 2>(a, exact, grid, items, st)
                         : p4_launch<64, M64>(a, exact, grid, items, st);
    case 128:
      return p.ct == 1   ? p4_launch<128, 1>(a, exact, grid, items, st)
             : p.ct == 2 ? p4_launch<128, 2>(a, exact, grid, items, st)
                         : p4_launch<128, M128>(a, exact, grid, items, st);
    default: return p4_launch<256, 1>(a, exact, grid, items, st);
  }
}
