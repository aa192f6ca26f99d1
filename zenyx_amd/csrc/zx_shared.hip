// zx_shared.hip -- attention for a batch whose sequences share pages: a group's common keys are
// read and multiplied once for the rows of all its sequences.  FP8 and 4-bit pages.
//
//   out_r = sum_t softmax(sm_scale q_r . K_t) V_t   over the keys t that row r sees
//
// Sequences [cu_group[g], cu_group[g + 1]) have their first shared_lens[g] positions on the same
// pages.  A row's keys are those of its group (positions below shared) and the others, on pages
// of its sequence alone: two sums with a running maximum each, (m, l, acc), merged at the end as
// the parts of a split sequence are.
//
// The group's keys: a tile is up to 16 CT columns (pairs of query row and head) of all the
// group's rows, so that a key that is read and converted serves many sequences; bound by the matrix
// products, conversions and exponentials of AttnWave once the columns are many, by the reads of
// the pages where they are few.  A sequence's own keys: its own rows' columns, bound by the reads.
// Both in one launch: blocks [0, n_pre) of a head take pieces of the groups' tiles, the others
// equal runs of the sequences' own units; how many of each, and how long the pieces are, every
// block finds from the lengths (on the device, so that a captured call may be replayed on
// others).  The pieces of one range of keys are neighbours, so that the tiles of a large group
// read a page while it is in the XCD's L2.
#include <algorithm>

#include "zx_attn_wave.h"
#include "zx_internal.h"

namespace zx {

constexpr uint32_t SH_UNIT = ATT_WAVES * AW_STEP;  // keys that a block takes per step

struct SharedArgs {
  const uint16_t *q;
  const int32_t *cu_q;  // NULL: a row per sequence
  const int32_t *bt, *seq_lens, *cu_group, *shared_lens;
  const uint8_t *pool;
  const float *scales;  // [2][n_kv_heads]; NULL (4 bits): ones
  uint16_t *out;
  int32_t *err;
  float *pre, *own;     // parts: [slot][n_q_heads][2 + D]
  void *table;
  int64_t n_pages, n_q, pre_slots;
  int32_t n_q_heads, n_kv_heads, page_size, max_blocks, n_seqs, n_groups, causal;
  int32_t most;            // rows of a sequence that are computed at most
  int32_t group, n_group;  // query heads per block, groups of them
  int32_t rows_p, rows_o;  // query rows per tile of a group, of a sequence
  int32_t n_rt;            // row tiles of a sequence at most
  int32_t n_run;           // blocks per group of heads
  uint32_t cap;            // positions that a block table holds
  uint32_t cost_p;         // of a group's unit, in quarters of an own unit
  uint32_t p_magic;
  int32_t p_shift;
  float sm_scale;
};

// What the merge needs to know: written once per call by a block of its own.
struct SharedSeq {
  uint64_t first;   // the sequence's first own unit
  uint32_t units;   // own units of each of its row tiles
  int32_t g;        // its group, -1: none
};
struct SharedGroup {
  uint64_t slot;    // of part 0 of its first row
  int64_t row0, rows;
  int64_t parts;    // 0: no shared keys
};
struct SharedTable {
  uint64_t *head;  // [2]: q, r of the deal
  SharedSeq *seq;
  SharedGroup *grp;
  __host__ __device__ SharedTable(void *at, int64_t n_seqs) {
    head = static_cast<uint64_t *>(at);
    seq = reinterpret_cast<SharedSeq *>(head + 2);
    grp = reinterpret_cast<SharedGroup *>(seq + n_seqs);
  }
  static size_t bytes(int64_t n_seqs, int64_t n_groups) {
    return 2 * sizeof(uint64_t) + (size_t)n_seqs * sizeof(SharedSeq) + (size_t)n_groups * sizeof(SharedGroup);
  }
};

__device__ __forceinline__ int64_t sh_row(const SharedArgs &a, int32_t b) {
  return a.cu_q ? max((int64_t)0, min((int64_t)a.cu_q[b], a.n_q)) : b;
}
// Shared positions of group g that are taken together: whole tiles of 16 tokens (what is left is
// read through each sequence's own table, which has it too).
__device__ __forceinline__ uint32_t sh_len(const SharedArgs &a, int32_t g) {
  const int32_t n = a.shared_lens[g];
  return n > 0 ? min((uint32_t)n, a.cap) & ~(uint32_t)(K4_TOK - 1) : 0u;
}
struct ShGroup {
  int32_t first, last;  // sequences
  int64_t row0, rows;
  uint32_t len, units, tiles;
  __device__ __forceinline__ ShGroup(const SharedArgs &a, int32_t g) {
    first = min(max(a.cu_group[g], 0), a.n_seqs);
    last = min(max(a.cu_group[g + 1], first), a.n_seqs);
    row0 = first < last ? sh_row(a, first) : 0;
    rows = first < last ? max((int64_t)0, sh_row(a, last) - row0) : 0;
    len = rows ? sh_len(a, g) : 0u;
    units = (len + (SH_UNIT - 1)) / SH_UNIT;
    tiles = units ? (uint32_t)((rows + a.rows_p - 1) / a.rows_p) : 0u;
  }
};
// The group of sequence b: the last one that begins at it or before, if it reaches b.
__device__ __forceinline__ int32_t sh_group_of(const SharedArgs &a, int32_t b) {
  int32_t lo = 0, hi = a.n_groups - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) >> 1;
    if (a.cu_group[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return a.n_groups > 0 && a.cu_group[lo] <= b && b < a.cu_group[lo + 1] ? lo : -1;
}
struct ShSeq {
  int64_t row0;
  int32_t rows, g;
  uint32_t keys, from;  // keys there are, and the first that is not the group's
  __device__ __forceinline__ uint32_t units() const { return keys > from ? (keys - from + (SH_UNIT - 1)) / SH_UNIT : 0u; }
  __device__ __forceinline__ uint32_t tiles(const SharedArgs &a) const { return (uint32_t)((rows + a.rows_o - 1) / a.rows_o); }
};
__device__ __forceinline__ ShSeq sh_seq(const SharedArgs &a, int32_t b, int32_t &e) {
  ShSeq s;
  s.row0 = b;
  s.rows = 1;
  if (a.cu_q) {
    const int64_t lo = a.cu_q[b], hi = a.cu_q[b + 1];
    if (lo < 0 || hi > a.n_q || hi - lo > a.most) e |= ZX_KERR_POS_RANGE;
    s.row0 = lo;
    s.rows = lo < 0 ? 0 : (int32_t)max((int64_t)0, min(min(hi, a.n_q) - lo, (int64_t)a.most));
  }
  const int32_t len = a.seq_lens[b];
  if (len > 0 && (uint32_t)len > a.cap) e |= ZX_KERR_POS_RANGE;
  s.keys = len > 0 ? min((uint32_t)len, a.cap) : 0u;
  s.g = sh_group_of(a, b);
  s.from = s.g >= 0 ? sh_len(a, s.g) : 0u;
  return s;
}

// Sums over the block's threads (every thread gets them); lds: of 4 words per value.
template <int N> __device__ __forceinline__ void sh_sums(uint64_t (&v)[N], uint64_t (*lds)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v[i] += __shfl_xor(v[i], off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) lds[threadIdx.x >> 6][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lds[0][i] + lds[1][i] + lds[2][i] + lds[3][i];
}

// How a call is dealt.
constexpr int SH_CAND = 8;
struct ShPlan {
  uint32_t n_pre;     // blocks (per group of heads) for the groups' tiles
  uint64_t n_seg;     // pieces of them
  uint32_t piece;     // their units at most
  uint64_t q, r;      // own units per block, and how many blocks have one more
};
struct ShLds {
  uint64_t sums[ATT_WAVES][SH_CAND];
  uint64_t base, slot;
  int32_t found;
  // sequences [win, win + 256): what their runs need
  int64_t row0[ATT_THREADS];
  int32_t rows[ATT_THREADS];
  uint32_t keys[ATT_THREADS], from[ATT_THREADS];
};

__device__ __forceinline__ ShPlan sh_plan(const SharedArgs &a, ShLds &lds, int32_t &e) {
  ShPlan p;
  uint64_t pq[2] = {0, 0};
  for (int32_t g = threadIdx.x; g < a.n_groups; g += ATT_THREADS) {
    const ShGroup s(a, g);
    pq[0] += (uint64_t)s.units * s.tiles;
  }
  for (int32_t b = threadIdx.x; b < a.n_seqs; b += ATT_THREADS) {
    const ShSeq s = sh_seq(a, b, e);
    pq[1] += (uint64_t)s.units() * s.tiles(a);
  }
  sh_sums<2>(pq, reinterpret_cast<uint64_t(*)[2]>(lds.sums));
  const uint64_t P = pq[0], Q = pq[1], n = (uint64_t)a.n_run;
  // blocks in the proportion of the work
  const float share = (float)P * (float)a.cost_p / ((float)P * (float)a.cost_p + 4.0f * (float)Q);
  p.n_pre = P == 0 ? 0u : Q == 0 ? (uint32_t)n : (uint32_t)max(1, min((int)n - 1, (int)((float)n * share + 0.5f)));
  p.piece = 1;
  p.n_seg = 0;
  if (p.n_pre) {
    // A piece of L units at most costs L and about 3 more (its start, its part of the merge); of a
    // few lengths the one with which the last block ends first.
    const uint64_t ideal = (P + p.n_pre - 1) / p.n_pre;
    uint32_t len[SH_CAND];
    uint64_t segs[SH_CAND];
#pragma unroll
    for (int k = 0; k < SH_CAND; ++k) {
      constexpr int EIGHTHS[SH_CAND] = {4, 8, 9, 10, 12, 16, 24, 32};
      len[k] = (uint32_t)min((uint64_t)0x40000000u, (ideal * EIGHTHS[k] + 7) / 8);
      segs[k] = 0;
    }
    for (int32_t g = threadIdx.x; g < a.n_groups; g += ATT_THREADS) {
      const ShGroup s(a, g);
#pragma unroll
      for (int k = 0; k < SH_CAND; ++k) segs[k] += (uint64_t)((s.units + len[k] - 1) / len[k]) * s.tiles;
    }
    sh_sums<SH_CAND>(segs, lds.sums);
    uint64_t best = ~0ull;
#pragma unroll
    for (int k = 0; k < SH_CAND; ++k) {
      const uint64_t t = (segs[k] + p.n_pre - 1) / p.n_pre * (len[k] + 3);
      if (t <= best) best = t, p.piece = len[k], p.n_seg = segs[k];
    }
    if (Q == 0) p.n_pre = (uint32_t)n;
    else if (p.n_seg < p.n_pre) p.n_pre = (uint32_t)p.n_seg;  // (the others take own units)
  }
  const uint64_t rest = n - p.n_pre;
  p.q = rest ? Q / rest : 0;
  p.r = rest ? Q % rest : 0;
  return p;
}

// Inclusive sum over the block's threads of v, and the sum of all; every thread calls it.
__device__ __forceinline__ uint64_t sh_scan(uint64_t v, uint64_t &all, ShLds &lds, int at) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t y = __shfl_up(v, off, 64);
    if (lane >= off) v += y;
  }
  __syncthreads();
  if (lane == 63) lds.sums[wave][at] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < ATT_WAVES; ++w) {
    if (w < wave) v += lds.sums[w][at];
    all += lds.sums[w][at];
  }
  return v;
}

// The group of piece `seg`: its number, its first piece and its first slot (found: -1 none).
__device__ __forceinline__ void sh_find_group(const SharedArgs &a, uint32_t piece, uint64_t seg, ShLds &lds) {
  uint64_t segs = 0, slots = 0;
  __syncthreads();
  if (threadIdx.x == 0) lds.found = -1;
  for (int32_t g0 = 0; g0 < a.n_groups; g0 += ATT_THREADS) {  // uniform
    const int32_t g = g0 + threadIdx.x;
    uint64_t n = 0, rows = 0, all_n, all_rows;
    if (g < a.n_groups) {
      const ShGroup s(a, g);
      const uint64_t parts = (s.units + piece - 1) / piece;
      n = parts * s.tiles;
      rows = parts * (uint64_t)s.rows;
    }
    const uint64_t in = sh_scan(n, all_n, lds, 0), ir = sh_scan(rows, all_rows, lds, 1);
    if (segs + in > seg && segs + in - n <= seg) {
      lds.found = g;
      lds.base = segs + in - n;
      lds.slot = slots + ir - rows;
    }
    segs += all_n;
    slots += all_rows;
    if (segs > seg) break;  // uniform
  }
  __syncthreads();
}

// Sequences [win, win + 256) into LDS.
__device__ __forceinline__ uint64_t sh_window(const SharedArgs &a, int32_t win, ShLds &lds) {
  const int32_t b = win + (int32_t)threadIdx.x;
  int32_t e = 0;
  ShSeq s = {};
  if (b < a.n_seqs) s = sh_seq(a, b, e);
  __syncthreads();
  lds.row0[threadIdx.x] = s.row0;
  lds.rows[threadIdx.x] = s.rows;
  lds.keys[threadIdx.x] = s.keys;
  lds.from[threadIdx.x] = s.from;
  __syncthreads();
  return b < a.n_seqs ? (uint64_t)s.units() * s.tiles(a) : 0;
}
// The sequence of own unit u: its number and first unit, with its window in LDS; returns the window's first.
__device__ __forceinline__ int32_t sh_find_seq(const SharedArgs &a, uint64_t u, ShLds &lds) {
  uint64_t before = 0;
  int32_t win = 0;
  for (;; win += ATT_THREADS) {  // uniform; u is below the sum of all
    const uint64_t n = sh_window(a, win, lds);
    uint64_t all;
    const uint64_t in = sh_scan(n, all, lds, 0);
    if (before + in > u && before + in - n <= u) {
      lds.found = win + (int32_t)threadIdx.x;
      lds.base = before + in - n;
    }
    before += all;
    if (before > u || win + ATT_THREADS >= a.n_seqs) break;
  }
  __syncthreads();
  return win;
}

// The block of its own: the table.
__device__ __forceinline__ void sh_write_table(const SharedArgs &a, const ShPlan &p, ShLds &lds, int32_t &e) {
  const SharedTable t(a.table, a.n_seqs);
  if (threadIdx.x == 0) {
    t.head[0] = p.q;
    t.head[1] = p.r;
  }
  uint64_t before = 0;
  for (int32_t b0 = 0; b0 < a.n_seqs; b0 += ATT_THREADS) {  // uniform
    const int32_t b = b0 + threadIdx.x;
    ShSeq s = {};
    if (b < a.n_seqs) s = sh_seq(a, b, e);
    const uint32_t units = b < a.n_seqs ? s.units() : 0u;
    const uint64_t n = (uint64_t)units * s.tiles(a);
    uint64_t all;
    const uint64_t in = sh_scan(n, all, lds, 0);
    if (b < a.n_seqs) t.seq[b] = SharedSeq{before + in - n, units, s.g};
    before += all;
  }
  uint64_t slots = 0;
  for (int32_t g0 = 0; g0 < a.n_groups; g0 += ATT_THREADS) {  // uniform
    const int32_t g = g0 + threadIdx.x;
    uint64_t rows = 0, parts = 0, all;
    int64_t row0 = 0, n_rows = 0;
    if (g < a.n_groups) {
      const ShGroup s(a, g);
      // groups are in order, and none reaches beyond the sequences
      if (a.cu_group[g] < 0 || a.cu_group[g + 1] < a.cu_group[g] || a.cu_group[g + 1] > a.n_seqs) e |= ZX_KERR_POS_RANGE;
      if (s.first < s.last && a.shared_lens[g] > 0 && (uint32_t)a.shared_lens[g] > a.cap) e |= ZX_KERR_POS_RANGE;
      parts = s.tiles ? (s.units + p.piece - 1) / p.piece : 0;
      rows = parts * (uint64_t)s.rows;
      row0 = s.row0;
      n_rows = s.rows;
    }
    const uint64_t ir = sh_scan(rows, all, lds, 0);
    if (g < a.n_groups) t.grp[g] = SharedGroup{slots + ir - rows, row0, n_rows, (int64_t)parts};
    slots += all;
  }
}

// Up to 16 CT columns of a head group on keys [t_begin, t_end): rows row0 .. row0 + n_rows of q; lim(r):
// keys below it count for row r; part(r): where row r's parts are (of its first head).
template <class F, int CT, bool EXACT, int POLICY, class Lim, class Part>
__device__ __forceinline__ void sh_segment(const SharedArgs &a, const AttnPages &pg, float scale, int G, int hq0,
                                           int64_t row0, int n_rows, uint32_t t_begin, uint32_t t_end,
                                           uint8_t (&lds)[ATT_WAVES][AttnLds<F::DIM>::WAVE],
                                           float (&sm_m)[ATT_WAVES][AW_COLS], float (&sm_l)[ATT_WAVES][AW_COLS],
                                           int32_t &e, Lim lim, Part part) {
  constexpr int D = F::DIM;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  AttnWave<F, CT, EXACT, POLICY> w(scale, lds[wave]);
  const int cols = n_rows * G;
  bool all = true;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = 16 * ct + w.n, r = c / G;
    const bool live = c < cols;
    w.lim[ct] = live ? min(t_end, lim(r)) : t_end;
    all &= w.lim[ct] == t_end;
    w.load_q(ct, a.q + ((row0 + (live ? r : 0)) * a.n_q_heads + hq0 + (live ? c - r * G : 0)) * D, live);
  }
  // (0: every step is masked)
  w.lim_all = __builtin_amdgcn_ballot_w64(!all) ? 0u : t_end;
  w.clear();
  const uint32_t t0 = t_begin + (uint32_t)wave * AW_STEP;
  if (t0 < t_end) w.run(pg, t0, t_end, ATT_WAVES * AW_STEP);
  e |= w.e;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (16 * ct >= cols) break;  // block-uniform
    w.spill(ct, cols - 16 * ct, sm_m[wave], sm_l[wave]);
    __syncthreads();
    const int c = 16 * ct + AttnEnd<D>::column();
    if (c < cols) {
      const AttnEnd<D> end(sm_m, sm_l, lds);
      const int r = c / G;
      end.store_part(part(r) + (int64_t)(hq0 + (c - r * G)) * (2 + D));
    }
    __syncthreads();
  }
}

__host__ __device__ constexpr int sh_per_cu(int D, int CT) { return D * CT > 128 ? 2 : CT > 1 ? 3 : 4; }

template <class F, int CT, int CTO, bool EXACT>
__global__ void __launch_bounds__(ATT_THREADS, sh_per_cu(F::DIM, CT)) paged_shared_kernel(SharedArgs a) {
  constexpr int D = F::DIM;
  __shared__ __attribute__((aligned(16))) uint8_t lds[ATT_WAVES][AttnLds<D>::WAVE];
  __shared__ float sm_m[ATT_WAVES][AW_COLS], sm_l[ATT_WAVES][AW_COLS];
  __shared__ ShLds sh;
  int32_t e = 0;
  const ShPlan p = sh_plan(a, sh, e);
  const uint32_t x = blockIdx.x / (uint32_t)a.n_group;
  if (x >= (uint32_t)a.n_run) {
    sh_write_table(a, p, sh, e);
    if (e && a.err) atomicOr(a.err, e);
    return;
  }
  e = 0;  // (reported by that block)
  const int y = (int)(blockIdx.x - x * (uint32_t)a.n_group);
  const int grp = a.n_q_heads / a.n_kv_heads, per_kv = a.n_group / a.n_kv_heads;
  const int h = y / per_kv, first = (y - h * per_kv) * a.group;
  const int G = min(a.group, grp - first), hq0 = h * grp + first;
  const int64_t head_bytes = (int64_t)(a.page_size / K4_TOK) * F::tile_bytes();
  AttnPages pg;
  pg.pool = a.pool;
  pg.n_pages = a.n_pages;
  pg.page_bytes = 2 * a.n_kv_heads * head_bytes;
  pg.head_off = h * head_bytes;
  pg.v_off = a.n_kv_heads * head_bytes;
  pg.page_size = (uint32_t)a.page_size;
  pg.p_magic = a.p_magic;
  pg.p_shift = a.p_shift;
  const float scale = a.sm_scale * ATT_LOG2E * (a.scales ? a.scales[h] : 1.0f);
  const int64_t row_part = (int64_t)a.n_q_heads * (2 + D);

  if (x < p.n_pre) {
    for (uint64_t seg = x; seg < p.n_seg; seg += p.n_pre) {
      sh_find_group(a, p.piece, seg, sh);
      const int32_t g = sh.found;
      if (g < 0) break;
      const ShGroup s(a, g);
      const uint32_t parts = (s.units + p.piece - 1) / p.piece;
      const uint32_t local = (uint32_t)(seg - sh.base), n = local / s.tiles, tile = local - n * s.tiles;
      const uint32_t t_begin = (uint32_t)((uint64_t)s.units * n / parts) * SH_UNIT;
      const uint32_t t_end = min(s.len, (uint32_t)((uint64_t)s.units * (n + 1) / parts) * SH_UNIT);
      const int64_t r0 = (int64_t)tile * a.rows_p;
      const int n_rows = (int)min((int64_t)a.rows_p, s.rows - r0);
      const uint64_t slot = sh.slot + (uint64_t)n * (uint64_t)s.rows + (uint64_t)r0;
      // (more only where groups overlap)
      if (slot + n_rows > (uint64_t)a.pre_slots) continue;
      pg.bt = a.bt + (int64_t)s.first * a.max_blocks;
      auto lim = [&](int r) -> uint32_t {  // the row's own sequence may be shorter than what its group shares
        const int64_t row = s.row0 + r0 + r;
        int32_t b = (int32_t)row;
        int64_t behind = 0;  // rows of the sequence after this one
        if (a.cu_q) {
          b = s.first;
          int32_t hi = s.last - 1;
          while (b < hi) {
            const int32_t mid = (b + hi + 1) >> 1;
            if (a.cu_q[mid] <= row) b = mid;
            else hi = mid - 1;
          }
          behind = a.causal ? (int64_t)a.cu_q[b + 1] - 1 - row : 0;
        }
        return (uint32_t)min(max((int64_t)a.seq_lens[b] - behind, (int64_t)0), (int64_t)a.cap);
      };
      sh_segment<F, CT, EXACT, 0>(a, pg, scale, G, hq0, s.row0 + r0, n_rows, t_begin, t_end, lds, sm_m, sm_l, e, lim,
                                  [&](int r) { return a.pre + (int64_t)(slot + r) * row_part; });
    }
  } else {
    const uint64_t xo = x - p.n_pre;
    uint64_t u = xo * p.q + min(xo, p.r);
    const uint64_t u_end = u + p.q + (xo < p.r ? 1 : 0);
    if (u < u_end) {
      int32_t win = sh_find_seq(a, u, sh);
      int32_t b = sh.found;
      uint64_t base = sh.base;
      while (u < u_end) {
        if (b >= a.n_seqs) break;
        if (b - win >= ATT_THREADS) {
          win = b;
          sh_window(a, win, sh);
        }
        ShSeq s;
        s.row0 = sh.row0[b - win];
        s.rows = sh.rows[b - win];
        s.keys = sh.keys[b - win];
        s.from = sh.from[b - win];
        const uint32_t units = s.units(), tiles = units ? s.tiles(a) : 0u;
        const uint64_t n = (uint64_t)units * tiles;
        if (u >= base + n) {
          base += n;
          ++b;
          continue;
        }
        const uint64_t local = u - base;
        const uint32_t rt = (uint32_t)(local / units), u0 = (uint32_t)(local - (uint64_t)rt * units);
        const uint32_t u1 = (uint32_t)min((uint64_t)units, u0 + (u_end - u));
        const int r0 = (int)rt * a.rows_o, n_rows = min(a.rows_o, s.rows - r0);
        // keys that row r of the tile sees
        auto lim = [&](int r) -> uint32_t {
          return a.causal ? (uint32_t)max((int64_t)s.keys - (s.rows - 1 - r0 - r), (int64_t)0) : s.keys;
        };
        const uint32_t t_begin = s.from + u0 * SH_UNIT;
        const uint32_t t_end = min(min(s.keys, s.from + u1 * SH_UNIT), lim(n_rows - 1));
        const uint64_t slot = (xo + (uint64_t)b * (uint64_t)a.n_rt + rt) * (uint64_t)a.rows_o;
        pg.bt = a.bt + (int64_t)b * a.max_blocks;
        sh_segment<F, CTO, EXACT, AW_STREAM>(a, pg, scale, G, hq0, s.row0 + r0, n_rows, t_begin, t_end, lds, sm_m, sm_l,
                                             e, lim, [&](int r) { return a.own + (int64_t)(slot + r) * row_part; });
        u += u1 - u0;
      }
    }
  }
  if (e && a.err) atomicOr(a.err, e);
}

// A channel of a row over its parts: att_combine_row's state, for lists one after the other.
struct ShCombine {
  float M = -INFINITY, L = 0.0f, A = 0.0f;
  __device__ __forceinline__ void add(const float *pp, int64_t step, int n, int d) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < n; base += 64) {
      const int cnt = min(64, n - base);
      const float *p0 = pp + (int64_t)base * step;
      const float ms = lane < cnt ? p0[lane * step] : -INFINITY;
      const float ls = lane < cnt ? p0[lane * step + 1] : 0.0f;
      float v[CB_U];
#pragma unroll
      for (int u = 0; u < CB_U; ++u) v[u] = p0[min(u, cnt - 1) * step + 2 + d];
      const float Mn = fmaxf(M, xrow_max(row16_max(ms)));
      const float alpha = __builtin_amdgcn_exp2f(M - Mn);  // (parts' maxima are finite: Mn is, after the first)
      const float w = __builtin_amdgcn_exp2f(ms - Mn);
      M = Mn;
      L = L * alpha + att_xrow_sum(group_sum<16>(w * ls));
      A *= alpha;
      for (int s = 0; s < cnt; s += CB_U) {
        float nx[CB_U];
        if (s + CB_U < cnt) {
#pragma unroll
          for (int u = 0; u < CB_U; ++u) nx[u] = p0[min(s + CB_U + u, cnt - 1) * step + 2 + d];
        }
#pragma unroll
        for (int u = 0; u < CB_U; ++u)
          if (s + u < cnt)
            A += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s + u)) * v[u];
#pragma unroll
        for (int u = 0; u < CB_U; ++u) v[u] = nx[u];
      }
    }
  }
};

// The rows: D threads per (row, head).
template <int D> __global__ void __launch_bounds__(256) shared_combine_kernel(SharedArgs a) {
  const int64_t at = (int64_t)blockIdx.x * (256 / D) + threadIdx.x / D;
  const int64_t row = at / a.n_q_heads;
  if (row >= a.n_q) return;
  const int hq = (int)(at - row * a.n_q_heads), d = threadIdx.x % D;
  const SharedTable t(a.table, a.n_seqs);
  int32_t b = (int32_t)row, i = 0;
  if (a.cu_q) {
    b = aw_seq_of(a.cu_q, a.n_seqs, (int32_t)row);
    const int64_t lo = a.cu_q[b], hi = a.cu_q[b + 1];
    // in no sequence, or not computed
    if (lo < 0 || row < lo || row >= hi || row - lo >= a.most) return;
    i = (int32_t)(row - lo);
  }
  const SharedSeq s = t.seq[b];
  const int64_t row_part = (int64_t)a.n_q_heads * (2 + D);
  ShCombine c;
  if (s.g >= 0) {
    const SharedGroup g = t.grp[s.g];
    const uint64_t slot = g.slot + (uint64_t)(row - g.row0);
    if (g.parts && slot + (uint64_t)((g.parts - 1) * g.rows) < (uint64_t)a.pre_slots)
      c.add(a.pre + (int64_t)slot * row_part + (int64_t)hq * (2 + D), g.rows * row_part, (int)g.parts, d);
  }
  if (s.units) {
    const AttnDeal<uint64_t> deal(t.head[0], t.head[1]);
    const int32_t rt = i / a.rows_o;
    const uint64_t u = s.first + (uint64_t)rt * s.units;
    const uint64_t xa = deal.run_of(u), xz = deal.run_of(u + s.units - 1);
    const int64_t slot = (int64_t)(xa + (uint64_t)b * (uint64_t)a.n_rt + (uint64_t)rt) * a.rows_o + (i - rt * a.rows_o);
    c.add(a.own + slot * row_part + (int64_t)hq * (2 + D), a.rows_o * row_part, (int)(xz - xa + 1), d);
  }
  const float sv = a.scales ? a.scales[a.n_kv_heads + hq / (a.n_q_heads / a.n_kv_heads)] : 1.0f;
  a.out[(row * a.n_q_heads + hq) * D + d] = (uint16_t)(pack_bf16(c.L == 0.0f ? 0.0f : c.A / c.L * sv, 0.0f) & 0xFFFFu);
}

}  // namespace zx

using namespace zx;

// Tiles of 16 columns that a block can hold.
static int sh_most_tiles(int D) { return D == 64 ? 4 : D == 128 ? 3 : 1; }

struct SharedHost {
  int ct, ct_own;
  int32_t group, n_group, rows_p, rows_o, n_rt;
  int64_t n_run, pre_slots, own_slots;
  size_t part_bytes, bytes;
};
static SharedHost sh_host(int64_t n_q, int32_t n_seqs, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                          int32_t head_dim, int32_t most) {
  SharedHost p;
  const int64_t grp = n_q_heads / n_kv_heads, subs = ceil_div(grp, AW_COLS);
  p.group = (int32_t)ceil_div(grp, subs);
  p.n_group = (int32_t)(n_kv_heads * subs);
  // column tiles per block: by the columns of a group on average, of a sequence at most
  const int tiles = sh_most_tiles(head_dim);
  const int64_t cols = ceil_div(n_q, std::max(n_groups, 1)) * p.group;
  p.ct = n_groups == 0 || cols <= 16 || tiles == 1 ? 1 : cols <= 32 ? 2 : tiles;
  const int64_t own = (int64_t)most * p.group;
  if (own > 16 && p.ct == 1 && tiles > 1) p.ct = own <= 32 ? 2 : tiles;
  p.ct_own = own <= 16 ? 1 : p.ct;
  p.rows_p = 16 * p.ct / p.group;
  p.rows_o = (int32_t)std::min<int64_t>(most, 16 * p.ct_own / p.group);
  p.n_rt = (int32_t)ceil_div(most, p.rows_o);
  p.n_run = std::max<int64_t>(2, (int64_t)sh_per_cu(head_dim, p.ct) * num_cus() / p.n_group);
  p.pre_slots = n_groups ? n_q + 2 * (p.n_run + 1) * p.rows_p : 0;
  p.own_slots = (p.n_run + (int64_t)n_seqs * p.n_rt) * p.rows_o;
  p.part_bytes = (size_t)((p.pre_slots + p.own_slots) * n_q_heads * (2 + head_dim)) * sizeof(float);
  p.bytes = p.part_bytes + SharedTable::bytes(n_seqs, n_groups);
  return p;
}
static bool sh_dims_ok(int64_t n_q, int32_t n_seqs, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                       int32_t head_dim, int32_t most) {
  return n_q > 0 && n_seqs > 0 && n_groups >= 0 && n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0 &&
         most > 0 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

extern "C" size_t zx_paged_attention_shared_workspace_bytes(int64_t n_q, int32_t n_seqs, int32_t n_groups,
                                                            int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                            int32_t max_q_per_seq) {
  if (!sh_dims_ok(n_q, n_seqs, n_groups, n_q_heads, n_kv_heads, head_dim, max_q_per_seq)) return 0;
  return sh_host(n_q, n_seqs, n_groups, n_q_heads, n_kv_heads, head_dim, max_q_per_seq).bytes;
}

template <class F, int CT, int CTO, bool EXACT> static int sh_launch(const SharedArgs &a, hipStream_t st) {
  paged_shared_kernel<F, CT, CTO, EXACT><<<(unsigned)(a.n_run * a.n_group + 1), ATT_THREADS, 0, st>>>(a);
  const int rc = check_launch("paged_shared");
  if (rc) return rc;
  shared_combine_kernel<F::DIM><<<(unsigned)ceil_div(a.n_q * a.n_q_heads, 256 / F::DIM), 256, 0, st>>>(a);
  return check_launch("shared_combine");
}

template <template <int> class Page, bool EXACT>
static int sh_call(const char *what, SharedArgs a, int32_t head_dim, int32_t max_q_per_seq, void *workspace,
                   size_t workspace_bytes, zx_stream_t stream) {
  int rc = k4_check(what, a.n_pages, a.n_kv_heads, head_dim, a.page_size);
  if (rc) return rc;
  ZX_REQUIRE(a.n_q >= 0 && max_q_per_seq >= 0 && a.n_q_heads > 0 && a.max_blocks > 0 && a.n_seqs > 0 && a.n_groups >= 0,
             "%s: sizes must be positive", what);
  ZX_REQUIRE(a.n_q_heads % a.n_kv_heads == 0, "%s: n_q_heads must be a multiple of n_kv_heads", what);
  ZX_REQUIRE((int64_t)a.max_blocks * a.page_size < (1LL << 31), "%s: block tables of 2^31 positions and more", what);
  ZX_REQUIRE(a.cu_q || a.n_q == a.n_seqs, "%s: without cu_q there is one row per sequence", what);
  if (a.n_seqs > 65535) return fail(ZX_ERR_UNSUPPORTED, "%s: more than 65535 sequences", what);
  ZX_REQUIRE(a.n_groups <= a.n_seqs, "%s: more groups than sequences", what);
  if (a.n_q == 0 || max_q_per_seq == 0) return ZX_OK;
  ZX_REQUIRE(a.q && a.pool && a.bt && a.seq_lens && a.out && (!a.n_groups || (a.cu_group && a.shared_lens)),
             "%s: null pointer", what);
  ZX_REQUIRE(aligned16(a.q) && aligned16(a.pool) && aligned16(a.out) && aligned16(workspace),
             "%s: q, pool, out and workspace must be 16-byte aligned", what);
  a.most = a.cu_q ? (int32_t)std::min<int64_t>(max_q_per_seq, a.n_q) : 1;
  const SharedHost p = sh_host(a.n_q, a.n_seqs, a.n_groups, a.n_q_heads, a.n_kv_heads, head_dim, a.most);
  if (a.n_q * a.n_q_heads >= (1LL << 31) || (int64_t)a.n_seqs * p.n_rt >= (1LL << 31))
    return fail(ZX_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (!workspace || workspace_bytes < p.bytes)
    return fail(ZX_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", what, workspace_bytes, p.bytes);
  a.pre = static_cast<float *>(workspace);
  a.own = a.pre + p.pre_slots * a.n_q_heads * (2 + head_dim);
  a.table = static_cast<uint8_t *>(workspace) + p.part_bytes;
  a.pre_slots = p.pre_slots;
  a.group = p.group;
  a.n_group = p.n_group;
  a.rows_p = p.rows_p;
  a.rows_o = p.rows_o;
  a.n_rt = p.n_rt;
  a.n_run = (int32_t)p.n_run;
  a.cap = (uint32_t)((int64_t)a.max_blocks * a.page_size);
  a.cost_p = p.ct == 1 ? 4 : p.ct == 2 ? 5 : 8;
  {  // magic division by the page size for positions below 2^31
    int sh = 0;
    while ((1LL << sh) < a.page_size) ++sh;
    a.p_shift = sh;
    a.p_magic = (uint32_t)(((1ULL << (31 + sh)) + (uint64_t)a.page_size - 1) / (uint64_t)a.page_size);
  }
  const hipStream_t st = as_stream(stream);
#define ZX_SH(D, CT, CTO) sh_launch<Page<D>, CT, CTO, EXACT>(a, st)
  switch (head_dim) {
    case 64:
      return p.ct == 1   ? ZX_SH(64, 1, 1)
             : p.ct == 2 ? (p.ct_own == 1 ? ZX_SH(64, 2, 1) : ZX_SH(64, 2, 2))
                         : (p.ct_own == 1 ? ZX_SH(64, 4, 1) : ZX_SH(64, 4, 4));
    case 128:
      return p.ct == 1   ? ZX_SH(128, 1, 1)
             : p.ct == 2 ? (p.ct_own == 1 ? ZX_SH(128, 2, 1) : ZX_SH(128, 2, 2))
                         : (p.ct_own == 1 ? ZX_SH(128, 3, 1) : ZX_SH(128, 3, 3));
    default: return ZX_SH(256, 1, 1);
  }
#undef ZX_SH
}

static SharedArgs sh_args(const uint16_t *q, int64_t n_q, const int32_t *cu_q, int32_t n_q_heads, const uint8_t *pool,
                          int64_t n_pages, int32_t n_kv_heads, int32_t page_size, const float *scales,
                          const int32_t *block_tables, int32_t max_blocks, const int32_t *seq_lens, int32_t n_seqs,
                          const int32_t *cu_group, const int32_t *shared_lens, int32_t n_groups, int32_t causal,
                          float sm_scale, uint16_t *out, int32_t *err) {
  SharedArgs a = {};
  a.q = q;
  a.cu_q = cu_q;
  a.bt = block_tables;
  a.seq_lens = seq_lens;
  a.cu_group = cu_group;
  a.shared_lens = shared_lens;
  a.pool = pool;
  a.scales = scales;
  a.out = out;
  a.err = err;
  a.n_pages = n_pages;
  a.n_q = n_q;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.page_size = page_size;
  a.max_blocks = max_blocks;
  a.n_seqs = n_seqs;
  a.n_groups = n_groups;
  a.causal = causal ? 1 : 0;
  a.sm_scale = sm_scale;
  return a;
}

extern "C" int zx_paged_attention_shared(const uint16_t *q, int64_t n_q, const int32_t *cu_q, int32_t n_q_heads,
                                         const uint8_t *pool, int64_t n_pages, int32_t n_kv_heads, int32_t head_dim,
                                         int32_t page_size, const float *scales, const int32_t *block_tables,
                                         int32_t max_blocks, const int32_t *seq_lens, int32_t n_seqs,
                                         const int32_t *cu_group, const int32_t *shared_lens, int32_t n_groups,
                                         int32_t max_q_per_seq, int32_t causal, float sm_scale, uint16_t *out,
                                         int32_t *err, void *workspace, size_t workspace_bytes, zx_stream_t stream) {
  clear_error();
  ZX_REQUIRE(scales, "paged_attention_shared: null pointer");
  return sh_call<Page8, false>("paged_attention_shared",
                               sh_args(q, n_q, cu_q, n_q_heads, pool, n_pages, n_kv_heads, page_size, scales, block_tables,
                                       max_blocks, seq_lens, n_seqs, cu_group, shared_lens, n_groups, causal, sm_scale, out,
                                       err),
                               head_dim, max_q_per_seq, workspace, workspace_bytes, stream);
}

extern "C" int zx_paged_attention4_shared(const uint16_t *q, int64_t n_q, const int32_t *cu_q, int32_t n_q_heads,
                                          const uint8_t *pool, int64_t n_pages, int32_t n_kv_heads, int32_t head_dim,
                                          int32_t page_size, const int32_t *block_tables, int32_t max_blocks,
                                          const int32_t *seq_lens, int32_t n_seqs, const int32_t *cu_group,
                                          const int32_t *shared_lens, int32_t n_groups, int32_t max_q_per_seq,
                                          int32_t causal, float sm_scale, uint16_t *out, int32_t *err, void *workspace,
                                          size_t workspace_bytes, zx_stream_t stream) {
  clear_error();
  return sh_call<Page4, true>("paged_attention4_shared",
                              sh_args(q, n_q, cu_q, n_q_heads, pool, n_pages, n_kv_heads, page_size, nullptr, block_tables,
                                      max_blocks, seq_lens, n_seqs, cu_group, shared_lens, n_groups, causal, sm_scale, out,
                                      err),
                              head_dim, max_q_per_seq, workspace, workspace_bytes, stream);
}
