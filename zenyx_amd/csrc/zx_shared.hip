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
// products, conversions and exponentials of AttnWave (of sh_wide: 128 columns, FP8 pages at D = 128) once
// the columns are many, by the reads of the pages where they are few.  A sequence's own keys: its own
// rows' columns, bound by the reads.
// Both in one launch: blocks [0, n_pre) of a head take pieces of the groups' tiles, the others
// equal runs of the sequences' own units; how many of each, and how long the pieces are, every
// block finds from the lengths (on the device, so that a captured call may be replayed on
// others).  The pieces of one range of keys are neighbours, so that the tiles of a large group
// read a page while it is in the XCD's L2.
#include <algorithm>

#include "zx_attn_tile.h"
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
  float cost_p;            // of a group's unit, in own units
  uint32_t p_magic;
  int32_t p_shift;
  float sm_scale;
};

// What the merge needs to know of a sequence: written once per call by a block of its own.
struct SharedSeq {
  uint32_t first;   // its first own unit
  uint32_t units;   // own units of each of its row tiles
  uint32_t parts;   // parts of its shared keys
  int32_t row0;     // the group's first row of q
  int64_t slot;     // of part 0 of its shared keys, for that row
  int64_t step;     // slots from one part to the next: the group's rows
};
struct SharedTable {
  uint32_t *head;  // [2]: q, r of the deal
  SharedSeq *seq;
  __host__ __device__ explicit SharedTable(void *at) {
    head = static_cast<uint32_t *>(at);
    seq = reinterpret_cast<SharedSeq *>(head + 4);
  }
  static size_t bytes(int64_t n_seqs) { return 4 * sizeof(uint32_t) + (size_t)n_seqs * sizeof(SharedSeq); }
};

// A value that is the same in all lanes, as a scalar.
__device__ __forceinline__ int32_t sh_uni(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t sh_uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ int64_t sh_uni(int64_t v) {
  return (int64_t)(((uint64_t)sh_uni((uint32_t)((uint64_t)v >> 32)) << 32) | sh_uni((uint32_t)v));
}

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
  int32_t all;          // rows that cu_q gives it, computed or not: row i is at position keys - all + i
  uint32_t keys, from;  // keys there are, and the first that is not the group's
  __device__ __forceinline__ uint32_t units() const { return keys > from ? (keys - from + (SH_UNIT - 1)) / SH_UNIT : 0u; }
  __device__ __forceinline__ uint32_t tiles(const SharedArgs &a) const { return (uint32_t)((rows + a.rows_o - 1) / a.rows_o); }
};
__device__ __forceinline__ ShSeq sh_seq(const SharedArgs &a, int32_t b, int32_t &e) {
  ShSeq s;
  s.row0 = b;
  s.rows = s.all = 1;
  if (a.cu_q) {
    const int64_t lo = a.cu_q[b], hi = a.cu_q[b + 1];
    if (lo < 0 || hi < lo || hi > a.n_q || hi - lo > a.most) e |= ZX_KERR_POS_RANGE;
    s.row0 = lo;
    s.rows = lo < 0 ? 0 : (int32_t)max((int64_t)0, min(min(hi, a.n_q) - lo, (int64_t)a.most));
    s.all = lo < 0 ? 0 : (int32_t)max((int64_t)0, hi - lo);
  }
  const int32_t len = a.seq_lens[b];
  if (len > 0 && (uint32_t)len > a.cap) e |= ZX_KERR_POS_RANGE;
  s.keys = len > 0 ? min((uint32_t)len, a.cap) : 0u;
  s.g = sh_group_of(a, b);
  s.from = s.g >= 0 ? sh_len(a, s.g) : 0u;
  return s;
}

template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t sh_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
// Inclusive sum over the wave's lanes.
__device__ __forceinline__ uint32_t sh_wave_scan(uint32_t v) {
  v += sh_dpp<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += sh_dpp<0x112, 0xF>(v);
  v += sh_dpp<0x114, 0xF>(v);
  v += sh_dpp<0x118, 0xF>(v);
  v += sh_dpp<0x142, 0xA>(v);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
  v += sh_dpp<0x143, 0xC>(v);
  return v;
}

// How a call is dealt.
constexpr int SH_CAND = 8;
constexpr int SH_STAGE = 256;  // sequences (and groups) whose lengths are kept in LDS
struct ShPlan {
  uint32_t n_pre;  // blocks (per group of heads) for the groups' tiles
  uint32_t n_seg;  // pieces of them
  uint32_t piece;  // their units at most
  uint32_t q, r;   // own units per block, and how many blocks have one more
};
struct ShLds {
  uint32_t sums[ATT_WAVES][SH_CAND];
  uint32_t base, slot;
  int32_t found;
  int32_t lens[SH_STAGE], shared[SH_STAGE], cu_q[SH_STAGE + 1], cu_group[SH_STAGE + 1];
};

// Sums over the block's threads, as scalars.
template <int N> __device__ __forceinline__ void sh_sums(uint32_t (&v)[N], ShLds &lds) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = sh_wave_scan(v[i]);
  __syncthreads();
  if ((threadIdx.x & 63) == 63)
#pragma unroll
    for (int i = 0; i < N; ++i) lds.sums[threadIdx.x >> 6][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = sh_uni(lds.sums[0][i] + lds.sums[1][i] + lds.sums[2][i] + lds.sums[3][i]);
}
// Inclusive sum over the block's threads of v, and the sum of all.
__device__ __forceinline__ uint32_t sh_scan(uint32_t v, uint32_t &all, ShLds &lds, int at) {
  const int wave = threadIdx.x >> 6;
  v = sh_wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds.sums[wave][at] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < ATT_WAVES; ++w) {
    const uint32_t n = lds.sums[w][at];
    if (w < wave) v += n;
    all += n;
  }
  all = sh_uni(all);
  return v;
}

// The lengths into LDS, all loads at once, where they fit: the searches below then cost no trip
// to memory each.
__device__ __forceinline__ void sh_stage(SharedArgs &a, ShLds &lds) {
  if (a.n_seqs > SH_STAGE) return;
  for (int i = threadIdx.x; i <= a.n_seqs; i += ATT_THREADS) {
    if (i < a.n_seqs) lds.lens[i] = a.seq_lens[i];
    if (a.cu_q) lds.cu_q[i] = a.cu_q[i];
    if (i < a.n_groups) lds.shared[i] = a.shared_lens[i];
    if (a.n_groups && i <= a.n_groups) lds.cu_group[i] = a.cu_group[i];
  }
  __syncthreads();
  a.seq_lens = lds.lens;
  if (a.cu_q) a.cu_q = lds.cu_q;
  a.shared_lens = lds.shared;
  a.cu_group = lds.cu_group;
}

__device__ __forceinline__ ShPlan sh_plan(const SharedArgs &a, ShLds &lds, int32_t &e) {
  ShPlan p;
  uint32_t pq[2] = {0, 0};  // (sums below 2^31: the host has seen to it)
  for (int32_t g = threadIdx.x; g < a.n_groups; g += ATT_THREADS) {
    const ShGroup s(a, g);
    pq[0] += s.units * s.tiles;
  }
  for (int32_t b = threadIdx.x; b < a.n_seqs; b += ATT_THREADS) {
    const ShSeq s = sh_seq(a, b, e);
    pq[1] += s.units() * s.tiles(a);
  }
  sh_sums<2>(pq, lds);
  const uint32_t P = pq[0], Q = pq[1], n = (uint32_t)a.n_run;
  // blocks in the proportion of the work
  const float wp = (float)P * a.cost_p, share = wp / (wp + (float)Q);
  p.n_pre = P == 0 ? 0u : Q == 0 ? n : (uint32_t)max(1, min((int)n - 1, (int)((float)n * share + 0.5f)));
  p.n_pre = sh_uni(p.n_pre);
  p.piece = 1;
  p.n_seg = 0;
  if (p.n_pre) {
    // A piece of L units at most costs L and about 3 more (its start, its part of the merge); of a
    // few lengths the one with which the last block ends first.
    const uint32_t ideal = (P + p.n_pre - 1) / p.n_pre;
    uint32_t len[SH_CAND], segs[SH_CAND];
#pragma unroll
    for (int k = 0; k < SH_CAND; ++k) {
      constexpr int EIGHTHS[SH_CAND] = {4, 8, 9, 10, 12, 16, 24, 32};
      len[k] = (uint32_t)(((uint64_t)ideal * EIGHTHS[k] + 7) / 8);
      segs[k] = 0;
    }
    for (int32_t g = threadIdx.x; g < a.n_groups; g += ATT_THREADS) {
      const ShGroup s(a, g);
#pragma unroll
      for (int k = 0; k < SH_CAND; ++k) segs[k] += (s.units + len[k] - 1) / len[k] * s.tiles;
    }
    sh_sums<SH_CAND>(segs, lds);
    uint64_t best = ~0ull;
#pragma unroll
    for (int k = 0; k < SH_CAND; ++k) {
      const uint64_t t = (uint64_t)((segs[k] + p.n_pre - 1) / p.n_pre) * (len[k] + 3);
      if (t <= best) best = t, p.piece = len[k], p.n_seg = segs[k];
    }
    p.piece = sh_uni(p.piece);
    p.n_seg = sh_uni(p.n_seg);
    if (Q && p.n_seg < p.n_pre) p.n_pre = p.n_seg;  // (the others take own units)
  }
  const uint32_t rest = n - p.n_pre;
  p.q = sh_uni(rest ? Q / rest : 0u);
  p.r = sh_uni(rest ? Q - p.q * rest : 0u);
  return p;
}

// The group of piece `seg`: its number (-1: none), its first piece and its first slot.
__device__ __forceinline__ int32_t sh_find_group(const SharedArgs &a, uint32_t piece, uint32_t seg, uint32_t &base,
                                                 uint32_t &slot, ShLds &lds) {
  uint32_t segs = 0, slots = 0;
  __syncthreads();
  if (threadIdx.x == 0) lds.found = -1;
  for (int32_t g0 = 0; g0 < a.n_groups; g0 += ATT_THREADS) {  // uniform
    const int32_t g = g0 + threadIdx.x;
    uint32_t n = 0, rows = 0, all_n, all_rows;
    if (g < a.n_groups) {
      const ShGroup s(a, g);
      const uint32_t parts = (s.units + piece - 1) / piece;
      n = parts * s.tiles;
      rows = parts * (uint32_t)s.rows;
    }
    const uint32_t in = sh_scan(n, all_n, lds, 0), ir = sh_scan(rows, all_rows, lds, 1);
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
  base = sh_uni(lds.base);
  slot = sh_uni(lds.slot);
  return sh_uni(lds.found);
}

// The sequence of own unit u, and its first unit.
__device__ __forceinline__ int32_t sh_find_seq(const SharedArgs &a, uint32_t u, uint32_t &base, ShLds &lds) {
  uint32_t before = 0;
  __syncthreads();
  if (threadIdx.x == 0) lds.found = a.n_seqs;
  for (int32_t b0 = 0; b0 < a.n_seqs; b0 += ATT_THREADS) {  // uniform
    const int32_t b = b0 + (int32_t)threadIdx.x;
    int32_t e = 0;
    uint32_t n = 0, all;
    if (b < a.n_seqs) {
      const ShSeq s = sh_seq(a, b, e);
      n = s.units() * s.tiles(a);
    }
    const uint32_t in = sh_scan(n, all, lds, 0);
    if (before + in > u && before + in - n <= u) {
      lds.found = b;
      lds.base = before + in - n;
    }
    before += all;
    if (before > u) break;
  }
  __syncthreads();
  base = sh_uni(lds.base);
  return sh_uni(lds.found);
}

// The block of its own: the table.
__device__ __forceinline__ void sh_write_table(const SharedArgs &a, const ShPlan &p, ShLds &lds, int32_t &e) {
  const SharedTable t(a.table);
  if (threadIdx.x == 0) {
    t.head[0] = p.q;
    t.head[1] = p.r;
  }
  uint32_t before = 0;
  for (int32_t b0 = 0; b0 < a.n_seqs; b0 += ATT_THREADS) {  // uniform
    const int32_t b = b0 + (int32_t)threadIdx.x;
    ShSeq s = {};
    if (b < a.n_seqs) s = sh_seq(a, b, e);
    const uint32_t units = b < a.n_seqs ? s.units() : 0u, n = units * s.tiles(a);
    uint32_t all;
    const uint32_t in = sh_scan(n, all, lds, 0);
    if (b < a.n_seqs) t.seq[b] = SharedSeq{before + in - n, units, 0u, 0, 0, 0};
    before += all;
  }
  uint32_t slots = 0;
  for (int32_t g0 = 0; g0 < a.n_groups; g0 += ATT_THREADS) {  // uniform
    const int32_t g = g0 + (int32_t)threadIdx.x;
    uint32_t rows = 0, parts = 0, all;
    int64_t row0 = 0, n_rows = 0;
    int32_t first = 0, last = 0;
    if (g < a.n_groups) {
      const ShGroup s(a, g);
      // groups are in order, and none reaches beyond the sequences
      if (a.cu_group[g] < 0 || a.cu_group[g + 1] < a.cu_group[g] || a.cu_group[g + 1] > a.n_seqs) e |= ZX_KERR_POS_RANGE;
      if (s.first < s.last && a.shared_lens[g] > 0 && (uint32_t)a.shared_lens[g] > a.cap) e |= ZX_KERR_POS_RANGE;
      parts = s.tiles ? (s.units + p.piece - 1) / p.piece : 0u;
      rows = parts * (uint32_t)s.rows;
      row0 = s.row0;
      n_rows = s.rows;
      first = s.first;
      last = s.last;
    }
    const uint32_t ir = sh_scan(rows, all, lds, 0);  // (and behind its barriers the entries above are written)
    const uint32_t slot = slots + ir - rows;
    if (parts && (uint64_t)slot + (uint64_t)parts * (uint64_t)n_rows <= (uint64_t)a.pre_slots)
      for (int32_t b = first; b < last; ++b) {
        t.seq[b].parts = parts;
        t.seq[b].row0 = (int32_t)row0;
        t.seq[b].slot = slot;
        t.seq[b].step = n_rows;
      }
    slots += all;
  }
}

// Up to 16 CT columns of a head group on keys [t_begin, t_end): columns c0 .. c0 + cols of those of
// rows row0 on; lim(r) (MASK): keys below it count for row r; part(r): where row r's parts are (of
// its first head).
template <class F, int CT, bool EXACT, int POLICY, bool MASK, class Lim, class Part>
__device__ __forceinline__ void sh_segment(const SharedArgs &a, const AttnPages &pg, float scale, int G, int hq0,
                                           int64_t row0, int c0, int cols, uint32_t t_begin, uint32_t t_end,
                                           uint8_t (&lds)[ATT_WAVES][AttnLds<F::DIM>::WAVE],
                                           float (&sm_m)[ATT_WAVES][AW_COLS], float (&sm_l)[ATT_WAVES][AW_COLS],
                                           int32_t &e, Lim lim, Part part) {
  constexpr int D = F::DIM;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  AttnWave<F, CT, EXACT, POLICY, MASK> w(scale, lds[wave]);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = c0 + 16 * ct + w.n, r = c / G;
    const bool live = 16 * ct + w.n < cols;
    if constexpr (MASK) w.lim[ct] = live ? min(t_end, lim(r)) : t_end;
    w.load_q(ct, a.q + ((row0 + (live ? r : 0)) * a.n_q_heads + hq0 + (live ? c - r * G : 0)) * D, live);
  }
  if constexpr (MASK) w.lim_all = 0;  // every step is masked
  w.clear();
  const uint32_t t0 = t_begin + (uint32_t)wave * AW_STEP;
  if (t0 < t_end) w.run(pg, t0, t_end, ATT_WAVES * AW_STEP);
  e |= w.e;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (16 * ct >= cols) break;  // block-uniform
    w.spill(ct, cols - 16 * ct, sm_m[wave], sm_l[wave]);
    __syncthreads();
    const int i = 16 * ct + AttnEnd<D>::column();
    if (i < cols) {
      const AttnEnd<D> end(sm_m, sm_l, lds);
      const int r = (c0 + i) / G;
      end.store_part(part(r) + (int64_t)(hq0 + (c0 + i - r * G)) * (2 + D));
    }
    __syncthreads();
  }
}

// A tile of 64 keys of a head in flight from FP8 pages to LDS: a thread has N pieces of 16 codes of K
// rows and as many of V, converts them on the way, and has its rows' page ids a tile ahead.
constexpr int SW_TILE = 64, SW_COLS = 32 * CR_WAVES;
template <int D> struct ShStage {
  static constexpr int PER_ROW = D / 16, N = SW_TILE * PER_ROW / CR_THREADS, STEP = CR_THREADS / PER_ROW;
  static_assert(N * CR_THREADS == SW_TILE * PER_ROW, "pieces dealt evenly");
  uint4 k[N], v[N];
  int32_t id[N];
  bool good[N];
  static __device__ __forceinline__ int row(int i) { return (int)threadIdx.x / PER_ROW + i * STEP; }
  static __device__ __forceinline__ int part() { return (int)threadIdx.x % PER_ROW; }
  // The pages of the thread's rows in the tile at t (positions from t_end on: of the last one).
  __device__ __forceinline__ void page(const AttnPages &pg, uint32_t t, uint32_t t_end) {
#pragma unroll
    for (int i = 0; i < N; ++i) id[i] = pg.bt[pg.page_of(min(t + (uint32_t)row(i), t_end - 1))];
  }
  __device__ __forceinline__ void load(const AttnPages &pg, uint32_t t, uint32_t t_end) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t at = min(t + (uint32_t)row(i), t_end - 1), in = at - pg.page_of(at) * pg.page_size;
      good[i] = id[i] >= 0 && id[i] < pg.n_pages;
      // (a bad page: the pool's first, whose codes are not used)
      const uint8_t *p = pg.pool + (int64_t)(good[i] ? id[i] : 0) * pg.page_bytes + pg.head_off + in * D + 16 * part();
      k[i] = *reinterpret_cast<const uint4 *>(p);
      v[i] = *reinterpret_cast<const uint4 *>(p + pg.v_off);
    }
  }
};
template <bool F16> __device__ __forceinline__ void sh_codes(uint4 c, att_u32x4 &lo, att_u32x4 &hi) {
  const uint32_t x[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    lo[n] = F16 ? aw_f16_of(x[n / 2], n & 1) : aw_bf16_of(x[n / 2], n & 1);
    hi[n] = F16 ? aw_f16_of(x[2 + n / 2], n & 1) : aw_bf16_of(x[2 + n / 2], n & 1);
  }
}

// Up to 128 columns on keys [t_begin, t_end) of FP8 pages, all of which every row sees.  The row sums add the
// weights before they are rounded (AttnWave: after): the rounding then moves a row by 2^-11 max|V|, half of
// what it does where both of the quotient's parts have it.  A wave has 32
// columns, and the four share tiles of 64 keys in LDS: a key is read and converted once per 128
// columns, where AttnWave's waves, with 48 columns and keys of their own, convert it for each 48 (D =
// 128, 64 sequences on 2,048 shared positions and 100-2,000 of their own 53 us, so 46; the other way
// D = 64, 12 heads, 64 sequences on 16,384 28 us, so 36, and 4 bits, whose second product is twice as long,
// 50 rows in 4 groups 74 us, so 92).
struct ShWideLds {
  static constexpr int D = 128;
  uint8_t k[2][SW_TILE * CrRowsOnly<D>::ROW];
  uint8_t v[2][CrLds<D, SW_TILE>::BYTES];
  uint8_t ok[2][4];  // are the 16-token quarters of a tile on pages that exist?
};
template <class Part>
__device__ __forceinline__ void sh_wide(const SharedArgs &a, const AttnPages &pg, float scale, int G, int hq0, int64_t row0,
                                        int cols, uint32_t t_begin, uint32_t t_end, ShWideLds &lds, int32_t &e, Part part) {
  constexpr int D = ShWideLds::D, KC = D / 16, DT = D / 32;
  using KRows = CrRowsOnly<D>;
  using T = CrF16;
  static_assert(T::BIAS == Page8<D>::BIAS, "parts of both kinds of segment are merged");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = 32 * wave + (lane & 31);
  const bool work = 32 * wave < cols, live = col < cols;
  const int r = live ? col / G : 0, hq = hq0 + (live ? col - r * G : 0);
  AttnScale qs(scale);
  att_u32x4 q[KC];
  {
    const uint16_t *p = a.q + ((row0 + r) * a.n_q_heads + hq) * D + 8 * (lane >> 5);
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      q[kc] = *reinterpret_cast<const att_u32x4 *>(p + 16 * kc);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[kc][i] = live ? (q[kc][i] ^ qs.flip) & qs.keep : 0u;
    }
  }
  cr_f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = cr_zero();
  float m = CR_NONE, top = CR_NONE, l = 0.0f;
  ShStage<D> st;
  auto load = [&](uint32_t t) {
    st.load(pg, t, t_end);
    if (t + SW_TILE < t_end) st.page(pg, t + SW_TILE, t_end);
  };
  auto store = [&](int buf, uint32_t t) {
#pragma unroll
    for (int i = 0; i < ShStage<D>::N; ++i) {
      const int row = ShStage<D>::row(i);
      // rows past the end, and those on bad pages, as zeros
      const bool there = st.good[i] && t + (uint32_t)row < t_end;
      const uint4 z = make_uint4(0u, 0u, 0u, 0u);
      att_u32x4 x, y;
      sh_codes<false>(there ? st.k[i] : z, x, y);
      uint8_t *k = KRows::at(lds.k[buf], row, 32 * ShStage<D>::part());
      *reinterpret_cast<att_u32x4 *>(k) = x;
      *reinterpret_cast<att_u32x4 *>(k + 16) = y;
      sh_codes<true>(there ? st.v[i] : z, x, y);
      *reinterpret_cast<att_u32x4 *>(cr_at<D>(lds.v[buf], row, 32 * ShStage<D>::part())) = x;
      *reinterpret_cast<att_u32x4 *>(cr_at<D>(lds.v[buf], row, 32 * ShStage<D>::part() + 16)) = y;
      if (ShStage<D>::part() == 0 && row % 16 == 0) {
        lds.ok[buf][row / 16] = st.good[i];
        if (!st.good[i] && t + (uint32_t)row < t_end) e |= ZX_KERR_PAGE_RANGE;
      }
    }
  };
  auto compute = [&](int buf, uint32_t t) {
    if (!work) return;
    const uint8_t *lk = KRows::at(lds.k[buf], lane & 31, 16 * (lane >> 5));
    uint8_t *lv = lds.v[buf];
    cr_f32x16 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = cr_zero();
#pragma unroll
      for (int kc = 0; kc < KC; ++kc)
        s[kt] = CrBf16::mfma(*reinterpret_cast<const att_u32x4 *>(lk + 32 * kt * KRows::ROW + 32 * kc), q[kc], s[kt]);
    }
    const uint32_t ok = *reinterpret_cast<const uint32_t *>(lds.ok[buf]);
    if (t + SW_TILE > t_end || __builtin_amdgcn_readfirstlane((int)ok) != 0x01010101) {  // uniform
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = 32 * kt + cr_row(i, lane);
          if (t + row >= t_end || !((ok >> (8 * (row / 16))) & 1u)) s[kt][i] = -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) mx = __builtin_elementwise_maximum(mx, s[i / 16][i % 16]);
    if (__builtin_amdgcn_ballot_w64(mx > top)) {
      const float m_new = fmaxf(m, cr_halves_max(mx) * qs.f - T::BIAS), alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      top = (m_new + (CR_LAZY + T::BIAS)) / qs.f;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      float x[16];
      att_u32x4 p[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], qs.f, -m));
        l += x[i];
      }
      cr_operands<T>(x, p);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = T::mfma(cr_cols<D>(lv, 2 * kt + c, dt, lane), p[c], o[dt]);
    }
  };
  if (t_begin < t_end) {
    st.page(pg, t_begin, t_end);
    load(t_begin);
    store(0, t_begin);
    __syncthreads();
    int buf = 0;
    for (uint32_t t = t_begin; t < t_end; t += SW_TILE, buf ^= 1) {
      if (t + SW_TILE < t_end) load(t + SW_TILE);
      compute(buf, t);
      if (t + SW_TILE < t_end) store(buf ^ 1, t + SW_TILE);
      __syncthreads();
    }
  }
  const float sum = cr_halves_sum(l);
  if (!live) return;
  float *pp = part(r) + (int64_t)hq * (2 + D);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; i += 2)
      *reinterpret_cast<float2 *>(pp + 2 + 32 * dt + cr_row(i, lane)) = make_float2(o[dt][i], o[dt][i + 1]);
  if (lane < 32) *reinterpret_cast<float2 *>(pp) = make_float2(m, sum);
}

// Tiles of 16 columns of a group that a block takes at most: by AttnWave what leaves two waves per
// SIMD, of FP8 pages at D = 128 SH_WIDE (128 columns) by sh_wide instead.
constexpr int SH_WIDE = SW_COLS / AW_COLS;
__host__ __device__ constexpr int sh_most_tiles(int bits, int D) {
  return D == 256 ? 1 : D == 64 ? 4 : bits == 8 ? SH_WIDE : 3;
}
// Blocks per CU by the registers, and (D = 128) by LDS.  (Four at D = 64 with one tile.  FP8 pages, where they
// spill 14 to 32 registers: 8 groups of 2 sequences on 8,000 shared positions, 12 heads, 34.2 against 28.7
// us, of 8 on 400 and up to 2,000 of their own 34.1 against 31.3, of 16 the other way, 47.6 against 52.1.  4
// bits, where none spill: of 2 on 8,000 30.0 against 28.1, of 8 on 400 and 1,000 of their own 30.5 against
// 27.0, one of 16 on 16,000 24.1 against 20.9, 8 of 16 on 4,000 and 300 the other way, 34.9 against 36.5.)
__host__ __device__ constexpr int sh_per_cu(int D, int CT) { return D * CT > 128 ? 2 : 3; }

// CTO: column tiles of a sequence's own keys.  ROWS: several rows per sequence.
template <class F, int CT, int CTO, bool EXACT, bool ROWS>
__global__ void __launch_bounds__(ATT_THREADS, sh_per_cu(F::DIM, CT)) paged_shared_kernel(SharedArgs a) {
  constexpr int D = F::DIM;
  struct Narrow {
    uint8_t lds[ATT_WAVES][AttnLds<D>::WAVE];
    float m[ATT_WAVES][AW_COLS], l[ATT_WAVES][AW_COLS];
  };
  union Lds {  // one segment after the other
    Narrow n;
    ShWideLds w;
  };
  __shared__ __attribute__((aligned(256))) uint8_t raw[CT == SH_WIDE ? sizeof(Lds) : sizeof(Narrow)];
  Lds &u_lds = *reinterpret_cast<Lds *>(raw);
  auto &lds = u_lds.n.lds;
  auto &sm_m = u_lds.n.m, &sm_l = u_lds.n.l;
  __shared__ ShLds sh;
  int32_t e = 0;
  sh_stage(a, sh);
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
    for (uint32_t seg = x; seg < p.n_seg; seg += p.n_pre) {
      uint32_t base, slot;
      const int32_t g = sh_find_group(a, p.piece, seg, base, slot, sh);
      if (g < 0) break;
      const ShGroup s(a, g);
      const uint32_t units = sh_uni(s.units), tiles = sh_uni(s.tiles), len = sh_uni(s.len);
      const int32_t b0 = sh_uni(s.first), b1 = sh_uni(s.last);
      const uint32_t parts = (units + p.piece - 1) / p.piece;
      const uint32_t n = (seg - base) / tiles, tile = (seg - base) - n * tiles;
      const uint32_t t_begin = (uint32_t)((uint64_t)units * n / parts) * SH_UNIT;
      const uint32_t t_end = min(len, (uint32_t)((uint64_t)units * (n + 1) / parts) * SH_UNIT);
      const uint32_t r0 = tile * (uint32_t)a.rows_p, all_rows = sh_uni((uint32_t)s.rows);
      const int n_rows = (int)min((uint32_t)a.rows_p, all_rows - r0);
      const int64_t row0 = sh_uni(s.row0) + r0;
      slot += n * all_rows + r0;
      // (more only where groups overlap)
      if ((int64_t)slot + n_rows > a.pre_slots) continue;
      pg.bt = a.bt + (int64_t)b0 * a.max_blocks;
      auto lim = [&](int r) -> uint32_t {  // the row's own sequence may be shorter than what its group shares
        const int64_t row = row0 + r;
        int32_t b = (int32_t)row;
        int64_t behind = 0;  // rows of the sequence after this one
        if (a.cu_q) {
          if (ROWS) {
            b = b0;
            int32_t hi = b1 - 1;
            while (b < hi) {
              const int32_t mid = (b + hi + 1) >> 1;
              if (a.cu_q[mid] <= row) b = mid;
              else hi = mid - 1;
            }
          } else {  // one row each is computed: sequences without one between them
            b = aw_seq_of(a.cu_q, a.n_seqs, (int32_t)row);
          }
          behind = a.causal ? (int64_t)a.cu_q[b + 1] - 1 - row : 0;
        }
        return (uint32_t)max(min((int64_t)a.seq_lens[b], (int64_t)a.cap) - behind, (int64_t)0);
      };
      auto part = [&](int r) { return a.pre + (int64_t)(slot + r) * row_part; };
      const int cols = n_rows * G;
      // every row sees all of the piece?  (Otherwise a tile of columns at a time.)
      bool all = true;
      for (int r = threadIdx.x & 63; r < n_rows; r += 64) all &= lim(r) >= t_end;
      const bool plain = !__builtin_amdgcn_ballot_w64(!all);
      if constexpr (CT == SH_WIDE) {
        if (plain) {
          sh_wide(a, pg, scale, G, hq0, row0, cols, t_begin, t_end, u_lds.w, e, part);
          continue;
        }
      } else if (plain) {
        sh_segment<F, CT, EXACT, 0, false>(a, pg, scale, G, hq0, row0, 0, cols, t_begin, t_end, lds, sm_m, sm_l, e, lim,
                                           part);
        continue;
      }
      for (int c0 = 0; c0 < cols; c0 += AW_COLS)
        sh_segment<F, 1, EXACT, 0, true>(a, pg, scale, G, hq0, row0, c0, min(AW_COLS, cols - c0), t_begin, t_end, lds, sm_m,
                                         sm_l, e, lim, part);
    }
  } else {
    const uint32_t xo = x - p.n_pre;
    uint32_t u = xo * p.q + min(xo, p.r);
    const uint32_t u_end = u + p.q + (xo < p.r ? 1 : 0);
    if (u < u_end) {
      uint32_t base;
      int32_t b = sh_find_seq(a, u, base, sh);
      while (u < u_end && b < a.n_seqs) {
        int32_t unused = 0;
        const ShSeq s = sh_seq(a, b, unused);
        const uint32_t units = sh_uni(s.units()), tiles = sh_uni(s.tiles(a));
        if (u >= base + units * tiles) {
          base += units * tiles;
          ++b;
          continue;
        }
        const uint32_t keys = sh_uni(s.keys), from = sh_uni(s.from);
        const int rows = sh_uni(s.rows), all = sh_uni(s.all);
        const uint32_t rt = (u - base) / units, u0 = (u - base) - rt * units;
        const uint32_t u1 = min(units, u0 + (u_end - u));
        const int r0 = (int)rt * a.rows_o, n_rows = min(a.rows_o, rows - r0);
        // keys that row r of the tile sees (one row: t_end below says it)
        auto lim = [&](int r) -> uint32_t {
          return a.causal ? (uint32_t)max((int64_t)keys - (all - 1 - r0 - r), (int64_t)0) : keys;
        };
        const uint32_t t_begin = from + u0 * SH_UNIT;
        const uint32_t t_end = min(min(keys, from + u1 * SH_UNIT), lim(n_rows - 1));
        const int64_t slot = ((int64_t)xo + (int64_t)b * a.n_rt + rt) * a.rows_o;
        pg.bt = a.bt + (int64_t)b * a.max_blocks;
        sh_segment<F, CTO, EXACT, AW_STREAM, ROWS>(a, pg, scale, G, hq0, sh_uni(s.row0) + r0, 0, n_rows * G, t_begin,
                                                   t_end, lds, sm_m, sm_l, e, lim,
                                                   [&](int r) { return a.own + (slot + r) * row_part; });
        u += u1 - u0;
      }
    }
  }
  if (e && a.err) atomicOr(a.err, e);
}

// A channel of a row over its parts: as att_combine_row merges them, from two lists.
struct ShParts {
  const float *p[2];  // part 0 of each list
  int64_t step[2];
  int n[2];
  __device__ __forceinline__ const float *at(int i) const {
    return i < n[0] ? p[0] + i * step[0] : p[1] + (i - n[0]) * step[1];
  }
};
__device__ __forceinline__ float sh_combine(const ShParts &parts, int d) {
  const int lane = threadIdx.x & 63, n = parts.n[0] + parts.n[1];
  float M = -INFINITY, L = 0.0f, A = 0.0f;
  for (int base = 0; base < n; base += 64) {
    const int cnt = min(64, n - base);
    const float2 ml = lane < cnt ? *reinterpret_cast<const float2 *>(parts.at(base + lane)) : make_float2(-INFINITY, 0.0f);
    float v[CB_U];
#pragma unroll
    for (int u = 0; u < CB_U; ++u) v[u] = parts.at(base + min(u, cnt - 1))[2 + d];
    const float Mn = fmaxf(M, xrow_max(row16_max(ml.x)));  // (parts' maxima are finite)
    const float alpha = __builtin_amdgcn_exp2f(M - Mn), w = __builtin_amdgcn_exp2f(ml.x - Mn);
    M = Mn;
    L = L * alpha + att_xrow_sum(group_sum<16>(w * ml.y));
    A *= alpha;
    for (int s = 0; s < cnt; s += CB_U) {
      float nx[CB_U];
      if (s + CB_U < cnt) {
#pragma unroll
        for (int u = 0; u < CB_U; ++u) nx[u] = parts.at(base + min(s + CB_U + u, cnt - 1))[2 + d];
      }
#pragma unroll
      for (int u = 0; u < CB_U; ++u)
        if (s + u < cnt) A += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s + u)) * v[u];
#pragma unroll
      for (int u = 0; u < CB_U; ++u) v[u] = nx[u];
    }
  }
  return L == 0.0f ? 0.0f : A / L;
}

// The rows: D threads per (row, head).
template <int D> __global__ void __launch_bounds__(256) shared_combine_kernel(SharedArgs a) {
  const int64_t at = (int64_t)blockIdx.x * (256 / D) + threadIdx.x / D;
  const int64_t row = at / a.n_q_heads;
  if (row >= a.n_q) return;
  const int hq = (int)(at - row * a.n_q_heads), d = threadIdx.x % D;
  const SharedTable t(a.table);
  int32_t b = (int32_t)row, i = 0;
  if (a.cu_q) {
    b = aw_seq_of(a.cu_q, a.n_seqs, (int32_t)row);
    const int64_t lo = a.cu_q[b], hi = a.cu_q[b + 1];
    // in no sequence, or not computed
    if (lo < 0 || row < lo || row >= hi || row - lo >= a.most) return;
    i = (int32_t)(row - lo);
  }
  const AttnDeal<uint32_t> deal(t.head[0], t.head[1]);
  const SharedSeq s = t.seq[b];
  const int64_t row_part = (int64_t)a.n_q_heads * (2 + D), at_head = (int64_t)hq * (2 + D);
  ShParts c = {};
  // (a row outside its group's: cu_q out of order, which is flagged)
  if (s.parts && row >= s.row0 && row - s.row0 < s.step) {
    c.p[0] = a.pre + (s.slot + row - s.row0) * row_part + at_head;
    c.step[0] = s.step * row_part;
    c.n[0] = (int)s.parts;
  }
  if (s.units) {
    const int32_t rt = i / a.rows_o;
    const uint32_t u = s.first + (uint32_t)rt * s.units;
    const uint32_t xa = deal.run_of(u), xz = deal.run_of(u + s.units - 1);
    const int64_t slot = ((int64_t)xa + (int64_t)b * a.n_rt + rt) * a.rows_o + (i - rt * a.rows_o);
    c.p[1] = a.own + slot * row_part + at_head;
    c.step[1] = a.rows_o * row_part;
    c.n[1] = (int)(xz - xa + 1);
  }
  const float sv = a.scales ? a.scales[a.n_kv_heads + hq / (a.n_q_heads / a.n_kv_heads)] : 1.0f;
  a.out[(row * a.n_q_heads + hq) * D + d] = (uint16_t)(pack_bf16(sh_combine(c, d) * sv, 0.0f) & 0xFFFFu);
}

}  // namespace zx

using namespace zx;

struct SharedHost {
  int ct, ct_own;
  int32_t group, n_group, rows_p, rows_o, n_rt;
  int64_t n_run, pre_slots, own_slots;
  size_t part_bytes, bytes;
};
static SharedHost sh_host(int bits, int64_t n_q, int32_t n_seqs, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                          int32_t head_dim, int32_t max_blocks, int32_t page_size, int32_t most) {
  SharedHost p;
  const int64_t grp = n_q_heads / n_kv_heads, subs = ceil_div(grp, AW_COLS);
  p.group = (int32_t)ceil_div(grp, subs);
  p.n_group = (int32_t)(n_kv_heads * subs);
  // columns per block: by those of a group on average, and of a sequence at most
  const int64_t cols = n_groups ? ceil_div(n_q, n_groups) * p.group : 0, own = (int64_t)most * p.group;
  const int tiles = sh_most_tiles(bits, head_dim);
  p.ct = tiles == 1 || cols <= 16 ? 1 : cols <= 32 ? 2 : tiles;
  if (own > 16 && p.ct == 1 && tiles > 1) p.ct = 2;
  p.ct_own = most == 1 || p.ct == 1 ? 1 : 2;
  p.rows_p = 16 * p.ct / p.group;
  p.rows_o = (int32_t)std::min<int64_t>(most, 16 * p.ct_own / p.group);
  p.n_rt = (int32_t)ceil_div(most, p.rows_o);
  // as many blocks as the chip holds, or as there can be units (768 blocks without one cost a call 4 us)
  const int64_t units = ceil_div((int64_t)max_blocks * page_size, SH_UNIT);
  const int64_t most_units = units * ((int64_t)n_seqs * p.n_rt + ceil_div(n_q, p.rows_p) + n_groups);
  p.n_run = std::max<int64_t>(2, std::min<int64_t>(sh_per_cu(head_dim, p.ct) * num_cus() / p.n_group, most_units));
  p.pre_slots = n_groups ? n_q + 2 * (p.n_run + 1) * p.rows_p : 0;
  p.own_slots = (p.n_run + (int64_t)n_seqs * p.n_rt) * p.rows_o;
  p.part_bytes = (size_t)((p.pre_slots + p.own_slots) * n_q_heads * (2 + head_dim)) * sizeof(float);
  p.bytes = p.part_bytes + SharedTable::bytes(n_seqs);
  return p;
}
static bool sh_dims_ok(int64_t n_q, int32_t n_seqs, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                       int32_t head_dim, int32_t most) {
  return n_q > 0 && n_seqs > 0 && n_groups >= 0 && n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0 &&
         most > 0 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

static size_t sh_bytes(int bits, int64_t n_q, int32_t n_seqs, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                       int32_t head_dim, int32_t page_size, int32_t max_blocks, int32_t most) {
  if (!sh_dims_ok(n_q, n_seqs, n_groups, n_q_heads, n_kv_heads, head_dim, most) || page_size <= 0 || max_blocks <= 0) return 0;
  return sh_host(bits, n_q, n_seqs, n_groups, n_q_heads, n_kv_heads, head_dim, max_blocks, page_size, most).bytes;
}
extern "C" size_t zx_paged_attention_shared_workspace_bytes(int64_t n_q, int32_t n_seqs, int32_t n_groups,
                                                            int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                            int32_t page_size, int32_t max_blocks, int32_t max_q_per_seq) {
  return sh_bytes(8, n_q, n_seqs, n_groups, n_q_heads, n_kv_heads, head_dim, page_size, max_blocks, max_q_per_seq);
}
extern "C" size_t zx_paged_attention4_shared_workspace_bytes(int64_t n_q, int32_t n_seqs, int32_t n_groups,
                                                             int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                             int32_t page_size, int32_t max_blocks,
                                                             int32_t max_q_per_seq) {
  return sh_bytes(4, n_q, n_seqs, n_groups, n_q_heads, n_kv_heads, head_dim, page_size, max_blocks, max_q_per_seq);
}

template <class F, int CT, int CTO, bool EXACT, bool ROWS> static int sh_launch(const SharedArgs &a, hipStream_t st) {
  paged_shared_kernel<F, CT, CTO, EXACT, ROWS><<<(unsigned)(a.n_run * a.n_group + 1), ATT_THREADS, 0, st>>>(a);
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
  constexpr int BITS = Page<64>::BITS;
  const SharedHost p = sh_host(BITS, a.n_q, a.n_seqs, a.n_groups, a.n_q_heads, a.n_kv_heads, head_dim, a.max_blocks,
                               a.page_size, a.most);
  if (a.n_q * a.n_q_heads >= (1LL << 31) || (int64_t)a.n_seqs * p.n_rt >= (1LL << 31))
    return fail(ZX_ERR_UNSUPPORTED, "%s: too many rows", what);
  // units are counted in 32 bits
  const int64_t most_units = ceil_div((int64_t)a.max_blocks * a.page_size, SH_UNIT);
  if ((int64_t)a.n_seqs * p.n_rt * most_units >= (1LL << 31) ||
      (ceil_div(a.n_q, p.rows_p) + a.n_groups) * most_units >= (1LL << 31) || p.pre_slots >= (1LL << 31))
    return fail(ZX_ERR_UNSUPPORTED, "%s: too many rows for block tables of so many positions", what);
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
  // A group's unit is bound by its products, an own one by its reads: up to 4 tiles of columns take about as
  // long as an own unit (50 rows of 4-bit pages in 4 groups on 4k-16k shared positions, a group's unit
  // counted for 2 / 1 / 0.75 own ones: 112 / 79 / 79 us), 128 columns three times that (128 sequences on
  // 32k shared positions, counted for 2 / 3 / 4: 132 / 125 / 124 us).
  a.cost_p = p.ct == SH_WIDE ? 3.0f : 1.0f;
  a.cap = (uint32_t)((int64_t)a.max_blocks * a.page_size);
  {  // magic division by the page size for positions below 2^31
    int sh = 0;
    while ((1LL << sh) < a.page_size) ++sh;
    a.p_shift = sh;
    a.p_magic = (uint32_t)(((1ULL << (31 + sh)) + (uint64_t)a.page_size - 1) / (uint64_t)a.page_size);
  }
  const hipStream_t st = as_stream(stream);
#define ZX_SH(D, CT, CTO) (a.most > 1 ? sh_launch<Page<D>, CT, CTO, EXACT, true>(a, st) : sh_launch<Page<D>, CT, 1, EXACT, false>(a, st))
  switch (head_dim) {
    case 64: return p.ct == 1 ? ZX_SH(64, 1, 1) : p.ct == 2 ? ZX_SH(64, 2, 2) : ZX_SH(64, sh_most_tiles(BITS, 64), 2);
    case 128: return p.ct == 1 ? ZX_SH(128, 1, 1) : p.ct == 2 ? ZX_SH(128, 2, 2) : ZX_SH(128, sh_most_tiles(BITS, 128), 2);
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
