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
// counts (matrix cores are busy 27% of a long call's time, vector units 48%).  64 x 32k
// positions, 2.3 GB of pages: 380 us, 6.0 TB/s; 16 x 1k-8k, 85 MB: 24 us.
#include <algorithm>

#include "zx_attn_wave.h"
#include "zx_internal.h"

namespace zx {

// Blocks per CU (waves per SIMD) by the registers of CT tiles of columns.
__host__ __device__ constexpr int a4_per_cu(int D, int CT) { return D * CT > 128 ? 2 : CT > 1 ? 3 : 4; }

// The queries of a call that has several rows per sequence (NULL cu_q: one each, at the end).
struct A4Rows {
  const int32_t *cu_q, *q_pos0;
  int32_t most;    // rows of a sequence that are computed
  int32_t causal;
  int64_t n_q;     // rows that there are
};

// Rows [lo, hi) of a sequence that are computed: at most `most`, and none outside [0, n_q).
__device__ __forceinline__ int32_t a4_rows(int64_t lo, int64_t hi, int64_t n_q, int64_t most, int32_t &e) {
  if (lo < 0 || hi > n_q || hi - lo > most) e |= ZX_KERR_POS_RANGE;
  return lo < 0 ? 0 : (int32_t)max((int64_t)0, min(min(hi, n_q) - lo, most));
}

// Sequences dealt in equal runs (att_locate).  Up to 16 CT columns: the (query row, head) pairs of
// one sequence and KV head's group.  g.group heads per block at most; the last group of a KV
// head may have fewer.
template <int D, int CT, bool EXACT, bool ROWS>
__global__ void __launch_bounds__(ATT_THREADS, a4_per_cu(D, CT))
paged_decode4_kernel(const uint16_t *__restrict__ q, AttnGeom g, A4Rows qr, const uint8_t *__restrict__ pool,
                     const int32_t *__restrict__ block_tables, const int32_t *__restrict__ seq_lens,
                     float *__restrict__ part, uint16_t *__restrict__ out, int32_t *err, void *table) {
  AttnRun run = att_locate(g, seq_lens, AttnTable(table, g.n_seqs), blockIdx.x);
  const int grp = g.n_q_heads / g.n_kv_heads;
  const int per_kv = g.n_group / g.n_kv_heads;  // groups of query heads per KV head
  const int h = run.y / per_kv, first = (run.y - h * per_kv) * g.group;
  const int G = min(g.group, grp - first);
  const int hq0 = h * grp + first;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t head_bytes = (int64_t)(g.page_size / K4_TOK) * k4_tile_bytes(D);
  AttnPages pg;
  pg.pool = pool;
  pg.n_pages = g.n_pages;
  pg.page_bytes = 2 * g.n_kv_heads * head_bytes;
  pg.head_off = h * head_bytes;
  pg.v_off = g.n_kv_heads * head_bytes;
  pg.page_size = (uint32_t)g.page_size;
  pg.p_magic = g.p_magic;
  pg.p_shift = g.p_shift;
  __shared__ __attribute__((aligned(16))) uint8_t lds[ATT_WAVES][AttnLds<D>::WAVE];
  __shared__ float sm_m[ATT_WAVES][AW_COLS], sm_l[ATT_WAVES][AW_COLS];
  AttnWave<Page4<D>, CT, EXACT> w(g.sm_scale * ATT_LOG2E, lds[wave]);
  // rows of sequence b that are computed, and the first one's number
  auto rows_of = [&](int b, int64_t &row0) -> int {
    row0 = b;
    if constexpr (!ROWS) return 1;
    row0 = qr.cu_q[b];
    return a4_rows(row0, qr.cu_q[b + 1], qr.n_q, qr.most, w.e);
  };
  auto zero_rows = [&](int b) {  // an empty sequence
    int64_t row0;
    const int n_rows = rows_of(b, row0);
    for (int i = threadIdx.x; i < n_rows * G * D; i += ATT_THREADS) {
      const int r = i / (G * D);
      out[((row0 + r) * g.n_q_heads + hq0) * D + (i - r * G * D)] = 0;
    }
  };
  if (g.whole && run.u == run.u_end && run.x < g.n_seqs) zero_rows(run.b);
  while (run.u < run.u_end) {
    const int b = run.b;
    const int32_t len = att_len(g, seq_lens, run);
    const uint32_t b_units = att_units(g, len);
    const uint32_t seg_end = (uint32_t)min(run.u_end - run.b_first, (uint64_t)b_units);
    const bool whole_seq = run.u == run.b_first && seg_end == b_units;
    const uint32_t t_begin = (uint32_t)(run.u - run.b_first) * g.unit;
    const uint32_t t_end = min(att_live_len(g, len), seg_end * g.unit);
    if (t_begin < t_end) {
      int64_t row0;
      const int cols = rows_of(b, row0) * G;
      // positions past the block table are not attended to, and flagged
      if (threadIdx.x == 0 && (int64_t)len > (int64_t)g.max_blocks * g.page_size) w.e |= ZX_KERR_POS_RANGE;
      pg.bt = block_tables + (int64_t)b * g.max_blocks;
      const bool causal = ROWS && qr.causal;
      const int64_t pos0 = causal ? qr.q_pos0[b] : 0;
      w.lim_all = causal ? (uint32_t)max((int64_t)0, min((int64_t)t_end, pos0 + 1)) : t_end;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int c = 16 * ct + w.n, r = ROWS ? c / G : 0;
        w.lim[ct] = causal ? (uint32_t)max((int64_t)0, min((int64_t)t_end, pos0 + r + 1)) : t_end;
        w.load_q(ct, q + ((row0 + r) * g.n_q_heads + hq0 + (c - r * G)) * D, c < cols);
      }
      w.clear();
      const uint32_t t0 = t_begin + (uint32_t)wave * AW_STEP;
      if (t0 < t_end) w.run(pg, t0, t_end, ATT_WAVES * AW_STEP);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        if (16 * ct >= cols) break;  // block-uniform
        w.spill(ct, cols - 16 * ct, sm_m[wave], sm_l[wave]);
        __syncthreads();
        const int c = 16 * ct + AttnEnd<D>::column();
        if (c < cols) {
          const AttnEnd<D> end(sm_m, sm_l, lds);
          const int r = ROWS ? c / G : 0, hq = hq0 + (c - r * G);
          if (whole_seq) end.store(out + ((row0 + r) * g.n_q_heads + hq) * D);
          else end.store_part(part + ((int64_t)(r * g.n_q_heads + hq) * ((int64_t)g.n_run + g.n_seqs) + run.x + b) * (2 + D));
        }
        __syncthreads();
      }
    }
    run.u = run.b_first + seg_end;
    run.b_first += b_units;
    ++run.b;
  }
  if (w.e && err) atomicOr(err, w.e);
}

// Pass 2 of a call with several rows per sequence: a block per (sequence, head), D threads per row.
template <int D>
__global__ void __launch_bounds__(1024)
decode4_rows_combine_kernel(const float *__restrict__ part, AttnGeom g, A4Rows qr, const int32_t *__restrict__ seq_lens,
                            uint16_t *__restrict__ out, int32_t *err, void *table) {
  const int b = (int)(blockIdx.x / (uint32_t)g.n_q_heads);
  const int hq = (int)(blockIdx.x - (uint32_t)b * (uint32_t)g.n_q_heads);
  int32_t x0, n_live, e = 0;
  att_live(g, seq_lens, table, b, x0, n_live);
  if (n_live == 1) return;
  const int64_t lo = qr.cu_q[b];
  const int32_t rows = a4_rows(lo, qr.cu_q[b + 1], qr.n_q, qr.most, e);
  // (a sequence without keys is met here alone)
  if (e && err && n_live == 0 && hq == 0 && threadIdx.x == 0) atomicOr(err, e);
  const int d = threadIdx.x % D;
  for (int r = threadIdx.x / D; r < rows; r += blockDim.x / D) {
    const float *pp = part + (((int64_t)r * g.n_q_heads + hq) * ((int64_t)g.n_run + g.n_seqs) + x0 + b) * (2 + D);
    out[((lo + r) * g.n_q_heads + hq) * D + d] = att_combine_row(pp, 2 + D, n_live, d, 1.0f);
  }
}

// Blocks of queries.  A block takes a tile of the (query row, head) columns of one sequence and KV
// head's group, and its four waves every fourth step of 32 keys, each with a running softmax of
// its own, merged at the end.  So no wave waits for another within the loop, K goes from memory
// to the operand without LDS, every conversion serves CT products, and a K/V byte read serves
// 16 CT columns: what a block reads is small, the pages have 4 bits.  Bound by the issue of the
// matrix products, the conversions and the exponentials together: 2 x 2,048 rows on 4k and 14k
// positions, 32/8 heads, D = 128, weights rounded to bf16, 724 us or 925 TFLOP/s, matrix cores busy
// 41% and vector units 52% of the time; with a second product for the weights' low halves 924 us,
// 46% and 60%.  A library product of 8,192^3 reaches 1,109.
// With few tiles a tile's keys are shared by up to n_split blocks, whose parts
// prefill4_combine_kernel merges.
struct Prefill4Args {
  const uint16_t *q;
  const int32_t *cu_q, *q_pos0, *bt, *kv_len;
  const uint8_t *pool;
  uint16_t *out;
  float *part;  // [item][split][16 CT columns][2 + D]
  int32_t *err;
  int64_t n_pages;
  int32_t n_q_heads, n_kv_heads, page_size, max_blocks, n_seqs, causal;
  int32_t group, n_group;  // heads per block, groups of them
  int32_t order;           // P4Order (one part per tile, up to 64 sequences)
  uint32_t slots;          // blocks that the chip holds
  int32_t rows;            // query rows per tile: 16 CT / group
  int32_t n_rt, n_split;   // row tiles per sequence, the most blocks per tile
  uint32_t n_items;        // tiles: n_rt * n_group * n_seqs
  int64_t max_q, n_q;      // rows of a sequence that are computed at most; rows of q
  uint32_t p_magic;
  int32_t p_shift;
  float sm_log2e;
};
constexpr uint32_t P4_UNIT = ATT_WAVES * AW_STEP;  // keys that a block takes per step

// Keys that the rows below row_end of a sequence at qpos0 can see.
__device__ __forceinline__ uint32_t p4_keys(const Prefill4Args &a, int32_t kv_len, int64_t qpos0, int64_t row_end) {
  const int64_t len = max((int64_t)0, min((int64_t)kv_len, (int64_t)a.max_blocks * a.page_size));
  return (uint32_t)(a.causal ? min(len, max((int64_t)0, qpos0 + row_end)) : len);  // below 2^31
}
// Parts of a tile with so many keys: at least P4_PART units each, at most n_split.  A part starts
// anew and is merged (2 x 128 rows on 2,000 and 500 positions, 32/8 heads, D = 128: two units 35
// us, four 29; 200 rows on 2,000, 12 heads, D = 64 19.9 / 16.9; the other way 64 rows on 1,000
// 16.6 / 18.8).
constexpr int P4_PART = 4;
__device__ __forceinline__ int p4_parts(const Prefill4Args &a, uint32_t keys) {
  return max(1, min(a.n_split, (int)((keys + P4_UNIT - 1) / P4_UNIT / P4_PART)));
}

// Up to 64 sequences, lane b holding sequence b: which come first, and whether a wave takes a tile
// by itself.  A tile that four waves share costs about 6 us of a block's time besides its steps
// (four starts, the merge), one of a wave's own 4 us of a wave's, but the launch then ends with
// whole tiles: a step is 1.8 us of a wave's time.  So by themselves if the tiles are many for
// their length: 7 times the tiles per block slot exceed the longest one's steps.  Weights of one
// rounding / carried to 2^-17: 4 x 2,048 new rows, 32/8 heads, D = 128, shared 231 / 264 us, alone
// 206 / 243; 9 x 227-455 rows, 32/8 heads, D = 64 35 / 39 and 24 / 28; 8 x 768 rows on 1,024 keys 139
// / 155 and 117 / 142; the other way 2 x 2,048 rows on 4k and 14k 719 / 922 and 773 / 989.
struct P4Order {
  int32_t lo, hi, len, pos0;
  int before;  // sequences before this lane's
  bool alone;
  __device__ __forceinline__ explicit P4Order(const Prefill4Args &a) : lo(0), hi(0), len(0), pos0(0), before(0) {
    const int lane = threadIdx.x & 63;
    if (lane < a.n_seqs) {
      lo = a.cu_q[lane];
      hi = a.cu_q[lane + 1];
      len = a.kv_len[lane];
      pos0 = a.q_pos0[lane];
    }
    int32_t e = 0;
    const int32_t rows = a4_rows(lo, hi, a.n_q, a.max_q, e);
    const uint32_t tiles = (uint32_t)((rows + a.rows - 1) / a.rows) * (uint32_t)a.n_group;
    const uint32_t steps = rows > 0 ? (p4_keys(a, len, pos0, rows) + AW_STEP - 1) / AW_STEP : 0u;
    uint64_t all = 0;
    uint32_t most = 0;
    for (int i = 0; i < a.n_seqs; ++i) {
      const int32_t other = __builtin_amdgcn_readlane(len, i);
      before += other > len || (other == len && i < lane);
      all += (uint32_t)__builtin_amdgcn_readlane((int)tiles, i);
      most = max(most, (uint32_t)__builtin_amdgcn_readlane((int)steps, i));
    }
    alone = 7 * all > (uint64_t)a.slots * most;
  }
};

template <int D, int CT, bool EXACT>
__global__ void __launch_bounds__(ATT_THREADS, a4_per_cu(D, CT)) paged_prefill4_kernel(Prefill4Args a) {
  // the sequence with the most keys first, its last row tiles first (under a causal mask they
  // see the most): the chip is left with short tiles at the end; a tile's parts next to each other
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t item = blockIdx.x / (uint32_t)a.n_split;
  const int split = (int)(blockIdx.x - item * (uint32_t)a.n_split);
  bool alone = false;  // every wave has a tile
  const uint32_t per_seq = (uint32_t)a.n_group * (uint32_t)a.n_rt;
  uint32_t s = item / per_seq;
  int b = (int)s;
  int32_t lo, hi, kv_len;
  int64_t pos0;
  if (a.order) {
    const P4Order o(a);
    alone = o.alone;
    if (alone) {
      item = blockIdx.x * ATT_WAVES + wave;
      s = item / per_seq;
    }
    if (item >= a.n_items) return;
    b = __ffsll((long long)__ballot((int)(threadIdx.x & 63) < a.n_seqs && o.before == (int)s)) - 1;
    lo = __builtin_amdgcn_readlane(o.lo, b);
    hi = __builtin_amdgcn_readlane(o.hi, b);
    kv_len = __builtin_amdgcn_readlane(o.len, b);
    pos0 = __builtin_amdgcn_readlane(o.pos0, b);
  } else {
    lo = a.cu_q[b];
    hi = a.cu_q[b + 1];
    kv_len = a.kv_len[b];
    pos0 = a.q_pos0[b];
  }
  const uint32_t rem = item - s * per_seq;
  const uint32_t rt_rev = rem / (uint32_t)a.n_group;
  const int y = (int)(rem - rt_rev * (uint32_t)a.n_group);
  const int grp = a.n_q_heads / a.n_kv_heads, per_kv = a.n_group / a.n_kv_heads;
  const int h = y / per_kv, first = (y - h * per_kv) * a.group;
  const int G = min(a.group, grp - first), hq0 = h * grp + first;
  int32_t e = 0;
  const int32_t rows = a4_rows(lo, hi, a.n_q, a.max_q, e);
  if (kv_len > (int64_t)a.max_blocks * a.page_size) e |= ZX_KERR_POS_RANGE;
  const int64_t row0 = ((int64_t)a.n_rt - 1 - rt_rev) * a.rows;
  const int n_rows = (int)max((int64_t)0, min((int64_t)a.rows, rows - row0));
  const uint32_t end = p4_keys(a, kv_len, pos0, row0 + n_rows);
  const int parts = p4_parts(a, end);
  if (n_rows == 0 || split >= parts) {  // block-uniform, or the wave's own
    if (e && a.err && (threadIdx.x & 63) == 0) atomicOr(a.err, e);
    return;
  }
  const uint32_t units = (end + P4_UNIT - 1) / P4_UNIT;  // below 2^24, and at most 64 parts
  const uint32_t t_begin = units * (uint32_t)split / (uint32_t)parts * P4_UNIT;
  const uint32_t t_end = min(end, units * (uint32_t)(split + 1) / (uint32_t)parts * P4_UNIT);
  const int64_t head_bytes = (int64_t)(a.page_size / K4_TOK) * k4_tile_bytes(D);
  AttnPages pg;
  pg.pool = a.pool;
  pg.bt = a.bt + (int64_t)b * a.max_blocks;
  pg.n_pages = a.n_pages;
  pg.page_bytes = 2 * a.n_kv_heads * head_bytes;
  pg.head_off = h * head_bytes;
  pg.v_off = a.n_kv_heads * head_bytes;
  pg.page_size = (uint32_t)a.page_size;
  pg.p_magic = a.p_magic;
  pg.p_shift = a.p_shift;
  __shared__ __attribute__((aligned(16))) uint8_t lds[ATT_WAVES][AttnLds<D>::WAVE];
  __shared__ float sm_m[ATT_WAVES][AW_COLS], sm_l[ATT_WAVES][AW_COLS];
  AttnWave<Page4<D>, CT, EXACT> w(a.sm_log2e, lds[wave]);
  w.e = e;
  const int cols = n_rows * G;
  const uint16_t *q = a.q + ((lo + row0) * a.n_q_heads + hq0) * D;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = 16 * ct + w.n, r = c / G;
    w.lim[ct] = a.causal ? (uint32_t)max((int64_t)0, min((int64_t)end, pos0 + row0 + r + 1)) : end;
    w.load_q(ct, q + ((int64_t)r * a.n_q_heads + (c - r * G)) * D, c < cols);
  }
  w.lim_all = a.causal ? (uint32_t)max((int64_t)0, min((int64_t)end, pos0 + row0 + 1)) : end;
  w.clear();
  const uint32_t t0 = t_begin + (alone ? 0u : (uint32_t)wave * AW_STEP);
  if (t0 < t_end) w.run(pg, t0, t_end, alone ? AW_STEP : ATT_WAVES * AW_STEP);
  if (alone) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = 16 * ct + w.n, r = c / G;
      const float sum = w.row_sum(ct);
      if (c < cols) w.store_row(ct, sum, a.out + ((lo + row0 + r) * a.n_q_heads + hq0 + (c - r * G)) * (int64_t)D);
    }
    if (w.e && a.err) atomicOr(a.err, w.e);
    return;
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {  // one tile of columns after the other
    if (16 * ct >= cols) break;      // block-uniform
    w.spill(ct, cols - 16 * ct, sm_m[wave], sm_l[wave]);
    __syncthreads();
    const int c = 16 * ct + AttnEnd<D>::column();
    if (c < cols) {
      const AttnEnd<D> end(sm_m, sm_l, lds);
      const int r = c / G;
      if (parts == 1) end.store(a.out + ((lo + row0 + r) * a.n_q_heads + hq0 + (c - r * G)) * (int64_t)D);
      else end.store_part(a.part + (((int64_t)item * a.n_split + split) * (16 * CT) + c) * (int64_t)(2 + D));  // (s is b)
    }
    __syncthreads();
  }
  if (w.e && a.err) atomicOr(a.err, w.e);
}

// Merges the parts of tiles that were cut: a block of D threads per (row, head).
template <int D>
__global__ void __launch_bounds__(D) prefill4_combine_kernel(Prefill4Args a, int32_t columns) {
  const uint32_t row_all = blockIdx.x / (uint32_t)a.n_q_heads;
  const int hq = (int)(blockIdx.x - row_all * (uint32_t)a.n_q_heads);
  const int b = aw_seq_of(a.cu_q, a.n_seqs, (int32_t)row_all);
  int32_t e = 0;
  const int64_t q_lo = a.cu_q[b], row = (int64_t)row_all - q_lo;
  const int64_t rows = a4_rows(q_lo, a.cu_q[b + 1], a.n_q, a.max_q, e);
  if (row < 0 || row >= rows) return;  // in no sequence, or not computed
  const int grp = a.n_q_heads / a.n_kv_heads, per_kv = a.n_group / a.n_kv_heads;
  const int h = hq / grp, sub = (hq - h * grp) / a.group, first = sub * a.group;
  const int G = min(a.group, grp - first);
  const int64_t rt = row / a.rows, row_end = min(rows, (rt + 1) * a.rows);
  const int parts = p4_parts(a, p4_keys(a, a.kv_len[b], a.q_pos0[b], row_end));
  if (parts == 1) return;  // its block has written the row
  const int64_t item = ((int64_t)b * a.n_rt + a.n_rt - 1 - rt) * a.n_group + h * per_kv + sub;
  const int c = (int)(row - rt * a.rows) * G + (hq - h * grp - first);
  const float *pp = a.part + (item * a.n_split * columns + c) * (int64_t)(2 + D);
  a.out[(int64_t)blockIdx.x * D + threadIdx.x] = att_combine_row(pp, (int64_t)columns * (2 + D), parts, threadIdx.x, 1.0f);
}

// Tiles of 16 columns that a block can hold: what leaves two waves per SIMD.  (With two at most, D
// = 128, weights rounded to bf16: 2 x 2,048 rows on 8,000 positions 806 us against 703, 8,192 rows
// from nothing 735 / 601; D = 64, 2 x 2,048 rows on 4k and 14k 472 / 439.)
constexpr int a4_most_tiles(int D) { return D == 64 ? 4 : D == 128 ? 3 : 1; }

}  // namespace zx

using namespace zx;

// Query heads per block: as few groups of at most 16 as there can be, of equal size but the last.
static int32_t a4_groups(int32_t grp) { return (int32_t)ceil_div(grp, AW_COLS); }

// When sequences are dealt whole.  In a graph, Hq 32 / Hkv 8, D = 128, in runs / whole: 64 x 100-600
// keys 17.9 / 15.1 us, 64 x 1,000-1,200 26 / 22, 128 x 1,000-1,200 44 / 38; the other way 16 x
// 1,000-1,200 14.9 / 17, 64 x 200-4k 36 / 46, 64 x 100-16k 102 / 158, 256 x 100-16k 410 / 447.
// Several rows per sequence, whose start costs more (4 rows, 64 x 200-4k 53 / 50, 128 x 200-4k
// 85 / 78; the other way 64 x 100-16k 133 / 150).  As many sequences as runs or more and none
// above 8 units: whole whatever their lengths, without the launches for the other way of
// dealing (128 x 100-600, 12 heads, D = 64, tables of 600: 22.5 us, without them 16.0).
constexpr AttnSlack A4_SLACK = {20, 2, 5, 8, 8}, A4_SLACK_ROWS = {20, 2, 12, 8, 32};
// Sequences in equal runs: one row each (columns <= 16), or as many rows as a block's columns hold.
static AttnRuns a4_plan(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_blocks,
                        int32_t page_size, int ct, const AttnSlack &slack) {
  const int64_t groups = (int64_t)n_kv_heads * a4_groups(n_q_heads / n_kv_heads);
  // at D = 128 three blocks per CU though four fit: 1 x 32k positions 20.4 us against 23.6, 4 x
  // 100-16k 19.2 against 21.7, 32 x 32k 199 against 197
  const int64_t resident = std::min(a4_per_cu(head_dim, ct), head_dim == 64 ? 4 : 3) * (int64_t)num_cus();
  return att_runs(n_seqs, groups, resident, P4_UNIT, max_blocks, page_size, slack);
}

static bool a4_dims_ok(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_blocks,
                       int32_t page_size) {
  return n_seqs > 0 && n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0 && max_blocks > 0 &&
         page_size > 0 && page_size % K4_TOK == 0 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

extern "C" size_t zx_paged_attention4_decode_workspace_bytes(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads,
                                                             int32_t head_dim, int32_t max_blocks, int32_t page_size) {
  if (!a4_dims_ok(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size)) return 0;
  return att_workspace_bytes(a4_plan(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, 1, A4_SLACK), n_seqs,
                             n_q_heads, head_dim);
}

// Launches the runs of a plan; part and table lie in the workspace.
template <int D, int CT, bool EXACT, bool ROWS>
static int a4_launch_runs(const AttnRuns &p, const AttnGeom &g, const A4Rows &qr, const uint16_t *q,
                          const uint8_t *pool, const int32_t *bt, const int32_t *lens, uint16_t *out, int32_t *err,
                          void *workspace, hipStream_t st) {
  float *part = static_cast<float *>(workspace);
  void *table = part + (int64_t)qr.most * g.n_q_heads * (p.n_run + g.n_seqs) * (2 + D);
  int rc = att_make_table(g, lens, table, st);
  if (rc) return rc;
  paged_decode4_kernel<D, CT, EXACT, ROWS><<<(unsigned)(p.n_blk * g.n_group), ATT_THREADS, 0, st>>>(
      q, g, qr, pool, bt, lens, part, out, err, table);
  if ((rc = check_launch("paged_decode4"))) return rc;
  if (!ROWS) return att_combine(part, g, nullptr, lens, out, table, st);
  if (g.whole) return ZX_OK;
  decode4_rows_combine_kernel<D><<<(unsigned)(g.n_seqs * g.n_q_heads), D * std::min(1024 / D, qr.most), 0, st>>>(
      part, g, qr, lens, out, err, table);
  return check_launch("decode4_rows_combine");
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
  ZX_REQUIRE(!workspace || aligned16(workspace), "paged_attention4_decode: workspace must be 16-byte aligned");
  const size_t need =
      zx_paged_attention4_decode_workspace_bytes(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size);
  if (!workspace || workspace_bytes < need)
    return fail(ZX_ERR_WORKSPACE, "paged_attention4_decode: workspace %zu < %zu bytes", workspace_bytes, need);
  const AttnRuns p = a4_plan(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, 1, A4_SLACK);
  AttnGeom g = att_geom(p, n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, n_pages, sm_scale);
  const int32_t grp = n_q_heads / n_kv_heads;
  g.group = (int32_t)ceil_div(grp, a4_groups(grp));
  g.n_group = n_kv_heads * a4_groups(grp);
  ZX_REQUIRE(p.n_blk * g.n_group < (1LL << 31), "paged_attention4_decode: too many sequences or heads");
  const A4Rows qr = {nullptr, nullptr, 1, 0, n_seqs};
  const hipStream_t st = as_stream(stream);
  switch (head_dim) {
    case 64: return a4_launch_runs<64, 1, true, false>(p, g, qr, q, pool, block_tables, seq_lens, out, err, workspace, st);
    case 128: return a4_launch_runs<128, 1, true, false>(p, g, qr, q, pool, block_tables, seq_lens, out, err, workspace, st);
    default: return a4_launch_runs<256, 1, true, false>(p, g, qr, q, pool, block_tables, seq_lens, out, err, workspace, st);
  }
}

struct Prefill4Plan {
  int ct;
  bool runs;  // one tile per sequence and head group: dealt in equal runs
  int32_t group, n_group, rows;
  int64_t n_rt, items, n_split;
  AttnRuns deal;
};
static Prefill4Plan p4_plan(int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_blocks,
                            int32_t page_size, int32_t n_seqs, int32_t max_q) {
  Prefill4Plan p;
  const int32_t grp = n_q_heads / n_kv_heads;
  const int most = a4_most_tiles(head_dim);
  p.group = (int32_t)ceil_div(grp, a4_groups(grp));
  p.n_group = n_kv_heads * a4_groups(grp);
  // column tiles per block, by the columns that a sequence can have at most
  const int64_t columns = (int64_t)max_q * p.group;
  p.ct = columns <= 16 || most == 1 ? 1 : columns <= 32 ? 2 : most;
  p.rows = 16 * p.ct / p.group;
  p.n_rt = ceil_div(max_q, p.rows);
  p.items = p.n_rt * p.n_group * n_seqs;
  p.deal = a4_plan(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, p.ct, A4_SLACK_ROWS);
  // parts of a tile where the tiles do not fill the chip
  const int64_t units = ceil_div((int64_t)max_blocks * page_size, P4_UNIT);
  const int64_t resident = (int64_t)a4_per_cu(head_dim, p.ct) * num_cus();
  p.runs = p.n_rt == 1 && p.items < 4 * resident;
  p.n_split = std::max<int64_t>(1, std::min<int64_t>({units / P4_PART, resident / p.items, 64}));
  return p;
}
static size_t p4_bytes(const Prefill4Plan &p, int32_t n_seqs, int32_t n_q_heads, int32_t head_dim, int32_t max_q) {
  if (p.runs)
    return (size_t)max_q * n_q_heads * (p.deal.n_run + n_seqs) * (2 + head_dim) * sizeof(float) +
           (n_seqs > 64 ? AttnTable::bytes(n_seqs, p.deal.n_run) : 0);
  return p.n_split > 1 ? (size_t)p.items * p.n_split * 16 * p.ct * (2 + head_dim) * sizeof(float) : 0;
}

extern "C" size_t zx_paged_attention4_prefill_workspace_bytes(int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                              int32_t page_size, int32_t max_blocks, int32_t n_seqs,
                                                              int32_t max_q_per_seq) {
  if (!a4_dims_ok(n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size) || max_q_per_seq <= 0) return 0;
  return p4_bytes(p4_plan(n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, n_seqs, max_q_per_seq), n_seqs,
                  n_q_heads, head_dim, max_q_per_seq);
}

template <int D, int CT>
static int p4_launch(const Prefill4Args &a, bool exact, unsigned rows, hipStream_t st) {
  const unsigned grid = a.n_items * (unsigned)a.n_split;
  // (one tile of columns: at D = 64 and 128 a sequence of at most 16, bound by the reads, where the
  // second product is free; at D = 256 every call: it has no form with one)
  if (CT == 1 || exact)
    paged_prefill4_kernel<D, CT, true><<<grid, ATT_THREADS, 0, st>>>(a);
  else if constexpr (CT > 1)
    paged_prefill4_kernel<D, CT, false><<<grid, ATT_THREADS, 0, st>>>(a);
  const int rc = check_launch("paged_prefill4");
  if (rc || a.n_split == 1) return rc;
  prefill4_combine_kernel<D><<<rows, D, 0, st>>>(a, 16 * CT);
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
  ZX_REQUIRE(!workspace || aligned16(workspace), "paged_attention4_prefill: workspace must be 16-byte aligned");
  const Prefill4Plan p = p4_plan(n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, n_seqs, max_q_per_seq);
  if (p.items * p.n_split >= (1LL << 31) || n_q * n_q_heads >= (1LL << 31) || p.deal.n_blk * p.n_group >= (1LL << 31))
    return fail(ZX_ERR_UNSUPPORTED, "paged_attention4_prefill: too many rows");
  const bool room = workspace && workspace_bytes >= p4_bytes(p, n_seqs, n_q_heads, head_dim, max_q_per_seq);
  const bool exact = flags & ZX_PREFILL_EXACT_P;
  const hipStream_t st = as_stream(stream);
  if (p.runs && room) {
    AttnGeom g = att_geom(p.deal, n_seqs, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, n_pages, sm_scale);
    g.group = p.group;
    g.n_group = p.n_group;
    const A4Rows qr = {cu_q, q_pos0, max_q_per_seq, causal ? 1 : 0, n_q};
#define ZX_A4_RUNS(D, CT, EX) \
  a4_launch_runs<D, CT, EX, true>(p.deal, g, qr, q, pool, block_tables, kv_len, out, err, workspace, st)
    switch (head_dim) {
      case 64:
        return p.ct == 1   ? ZX_A4_RUNS(64, 1, true)
               : p.ct == 2 ? (exact ? ZX_A4_RUNS(64, 2, true) : ZX_A4_RUNS(64, 2, false))
                           : (exact ? ZX_A4_RUNS(64, 4, true) : ZX_A4_RUNS(64, 4, false));
      case 128:
        return p.ct == 1   ? ZX_A4_RUNS(128, 1, true)
               : p.ct == 2 ? (exact ? ZX_A4_RUNS(128, 2, true) : ZX_A4_RUNS(128, 2, false))
                           : (exact ? ZX_A4_RUNS(128, 3, true) : ZX_A4_RUNS(128, 3, false));
      default: return ZX_A4_RUNS(256, 1, true);
    }
#undef ZX_A4_RUNS
  }
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
  a.max_q = max_q_per_seq;
  a.n_q = n_q;
  a.sm_log2e = sm_scale * ATT_LOG2E;
  a.n_split = room && !p.runs ? (int32_t)p.n_split : 1;
  a.order = a.n_split == 1 && n_seqs <= 64;
  a.slots = (uint32_t)(a4_per_cu(head_dim, p.ct) * num_cus());
  {
    int sh = 0;
    while ((1LL << sh) < page_size) ++sh;
    a.p_shift = sh;
    a.p_magic = (uint32_t)(((1ULL << (31 + sh)) + (uint64_t)page_size - 1) / (uint64_t)page_size);
  }
  a.n_items = (uint32_t)p.items;
  const unsigned rows = (unsigned)(n_q * n_q_heads);
  switch (head_dim) {
    case 64:
      return p.ct == 1   ? p4_launch<64, 1>(a, exact, rows, st)
             : p.ct == 2 ? p4_launch<64, 2>(a, exact, rows, st)
                         : p4_launch<64, 4>(a, exact, rows, st);
    case 128:
      return p.ct == 1   ? p4_launch<128, 1>(a, exact, rows, st)
             : p.ct == 2 ? p4_launch<128, 2>(a, exact, rows, st)
                         : p4_launch<128, 3>(a, exact, rows, st);
    default: return p4_launch<256, 1>(a, exact, rows, st);
  }
}
