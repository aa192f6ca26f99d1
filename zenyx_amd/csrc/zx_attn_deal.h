// zx_attn_deal.h -- how decode attention deals the positions of all sequences to its blocks,
// for 8-bit (zx_attention.hip) and 4-bit pages (zx_attention4.hip) alike: units of positions
// laid end to end, equal runs of them, and the merge of a run's segments.
#pragma once

#include <algorithm>

#include "zx_attn_common.h"

namespace zx {

constexpr int ATT_THREADS = 256;  // 4 waves
constexpr int ATT_WAVES = ATT_THREADS / 64;

struct AttnGeom {
  int32_t n_q_heads, n_kv_heads, head_dim, page_size, max_blocks, n_seqs;
  int32_t n_run;        // equal runs, one block per head group each
  uint32_t unit, cap;   // positions per unit (a power of two); positions a block table holds
  uint32_t tail, part, more;  // see att_take_whole
  int32_t whole;        // every sequence is taken whole: known to the host
  int32_t group, n_group;       // query heads per block; groups of them
  uint32_t p_magic;  // t / page_size = (t * p_magic) >> (31 + p_shift) for t < 2^31
  int32_t p_shift;
  int64_t n_pages;
  float sm_scale;
};

__device__ __forceinline__ uint32_t page_of(const AttnGeom &g, uint32_t t) {
  return (uint32_t)(((uint64_t)t * g.p_magic) >> (31 + g.p_shift));
}

// Positions of a sequence that are attended to (lengths are int32).
__device__ __forceinline__ uint32_t att_live_len(const AttnGeom &g, int32_t len) {
  return len > 0 ? min((uint32_t)len, g.cap) : 0u;
}
__device__ __forceinline__ uint32_t att_units(const AttnGeom &g, int32_t len) {
  return (att_live_len(g, len) + (g.unit - 1)) / g.unit;  // unit: a power of two
}

// The U units of all sequences dealt to n_run runs: run x takes q = U / n_run of them, the
// first r = U % n_run one more.  T: 32 bits where U fits.
template <typename T> struct AttnDeal {
  T q, r;
  __device__ AttnDeal(T q_, T r_) : q(q_), r(r_) {}
  __device__ T begin(T x) const { return x * q + min(x, r); }
  __device__ T run_of(T u) const { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; }
};

// Whole sequences instead of equal runs?  A run starts anew in every sequence that it touches
// (q, the first page ids, K and V one after the other: about as long as four units) and its
// parts are merged; whole sequences leave blocks idle while the longest one ends.  So: if the
// longest one has at most tail units beyond the lesser of part / 8 of an equal share and a share
// and `more` (a call whose longest sequence is within the tail needs no sums).  The figures are
// the kernels' (AttnSlack).
__device__ __forceinline__ bool att_take_whole(const AttnGeom &g, uint64_t most, uint64_t share) {
  return most <= g.tail + min(share * g.part / 8, share + g.more);
}

// Inclusive sum over the lanes below n (n <= 64, uniform).
__device__ __forceinline__ uint32_t att_scan(uint32_t v, int n) {
  const int lane = threadIdx.x & 63;
  for (int off = 1; off < n; off <<= 1) {
    const uint32_t y = __shfl_up(v, off, 64);
    if (lane >= off) v += y;
  }
  return v;
}

// More than 64 sequences: what every block needs to know, computed once by att_plan_kernel.
struct AttnTable {
  uint64_t *head;   // [4]: whole sequences?, q, r
  uint64_t *first;  // [n_seqs] a sequence's first unit
  int32_t *x0, *n_live;  // [n_seqs] the first run that holds a part of it, and how many do
  int32_t *run_b;        // [n_run] the sequence in which a run begins
  __host__ __device__ AttnTable(void *at, int64_t n_seqs) {
    head = static_cast<uint64_t *>(at);
    first = head + 4;
    x0 = reinterpret_cast<int32_t *>(first + n_seqs);
    n_live = x0 + n_seqs;
    run_b = n_live + n_seqs;
  }
  static size_t bytes(int64_t n_seqs, int64_t n_run) {
    return 4 * sizeof(uint64_t) + (size_t)n_seqs * (sizeof(uint64_t) + 2 * sizeof(int32_t)) +
           (size_t)n_run * sizeof(int32_t);
  }
};

// The run of block x: units [u, u_end), unit u in sequence b, whose first unit is b_first.
// All block-uniform; an empty run has u == u_end.  Up to 64 sequences every lane keeps one
// sequence's length, so that stepping to the next sequence reads no memory.
struct AttnRun {
  uint64_t u, u_end, b_first;
  int32_t b, lane_len;
  int32_t x, y;  // the run (or sequence) and the group of query heads
};
__device__ __forceinline__ int32_t att_len(const AttnGeom &g, const int32_t *seq_lens, const AttnRun &r) {
  return g.n_seqs <= 64 ? __builtin_amdgcn_readlane(r.lane_len, r.b) : seq_lens[r.b];
}
// Lane b's units, and how up to 64 sequences are dealt: whole, or units [begin(x), begin(x +
// 1)) to run x, where incl is the inclusive sum over the sequences.
struct AttnLanes {
  uint32_t n, incl = 0;
  bool whole;
  AttnDeal<uint32_t> deal;
  __device__ AttnLanes(const AttnGeom &g, int32_t lane_len) : n(att_units(g, lane_len)), deal(0, 0) {
    whole = __ballot(n > g.tail) == 0;
    if (whole) return;
    incl = att_scan(n, g.n_seqs);
    const uint32_t all = __builtin_amdgcn_readlane(incl, g.n_seqs - 1);
    deal = AttnDeal<uint32_t>(all / (uint32_t)g.n_run, all % (uint32_t)g.n_run);
    whole = __ballot(!att_take_whole(g, n, deal.q)) == 0;
  }
};
// Block `at` of a one-dimensional grid: the groups of a run (or sequence) are neighbours, so
// that blocks that read the same pages run together, and the blocks without one come last
// (between the others they left three quarters of the CUs idle).
__device__ __forceinline__ AttnRun att_locate(const AttnGeom &g, const int32_t *seq_lens, const AttnTable &t,
                                              uint32_t at) {
  AttnRun r;
  const int lane = threadIdx.x & 63;
  r.lane_len = lane < g.n_seqs ? seq_lens[lane] : 0;
  r.x = (int)(at / (uint32_t)g.n_group);
  r.y = (int)(at - (uint32_t)r.x * (uint32_t)g.n_group);
  const int x = r.x;
  r.b = x;
  r.u = r.u_end = r.b_first = 0;
  bool whole = g.whole;
  uint64_t q = 0, rem = 0;
  if (!whole && g.n_seqs <= 64) {  // every wave by itself
    const AttnLanes l(g, r.lane_len);
    whole = l.whole;
    if (!whole && x < g.n_run) {
      const uint32_t u = l.deal.begin((uint32_t)x), u_end = l.deal.begin((uint32_t)x + 1);
      r.u = u;
      r.u_end = u_end;
      const uint64_t after = __ballot(l.incl > u);  // sequences that end after u; the first holds it
      r.b = after ? __ffsll((long long)after) - 1 : 0;
      r.b_first = __builtin_amdgcn_readlane(l.incl - l.n, r.b);
    }
  } else if (!whole) {
    whole = t.head[0] != 0;
    q = t.head[1];
    rem = t.head[2];
    if (!whole && x < g.n_run) {
      const AttnDeal<uint64_t> deal(q, rem);
      r.u = deal.begin((uint64_t)x);
      r.u_end = deal.begin((uint64_t)x + 1);
      if (r.u < r.u_end) {
        r.b = t.run_b[x];
        r.b_first = t.first[r.b];
      }
    }
  }
  if (whole && x < g.n_seqs) r.u_end = __builtin_amdgcn_readfirstlane(att_units(g, att_len(g, seq_lens, r)));
  return r;
}

// Merges the block's four waves' (m, l, acc[G][D]) (in LDS, after a barrier) and stores the
// segment's rows: bf16 rows when the segment is its whole sequence (zeros when no position
// had a page), else partial x + b of the row's n_run + n_seqs (moving along the runs, x or
// b or both grow from one segment to the next, so x + b names a segment).
template <int D, int ROWS>
__device__ __forceinline__ void att_store(const AttnGeom &g, const float (&sm_m)[ATT_WAVES][ROWS],
                                          const float (&sm_l)[ATT_WAVES][ROWS], const float *const (&acc)[ATT_WAVES],
                                          float *part, uint16_t *out, int G, int hq0, int b, int x, bool whole,
                                          float sv) {
  for (int idx = threadIdx.x; idx < G * D; idx += ATT_THREADS) {
    const int j = idx / D, d = idx % D;
    float M = sm_m[0][j];
#pragma unroll
    for (int w = 1; w < ATT_WAVES; ++w) M = fmaxf(M, sm_m[w][j]);
    float a = 0.0f, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < ATT_WAVES; ++w) {
      const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm_m[w][j] - M);
      a += f * acc[w][j * D + d];
      ll += f * sm_l[w][j];
    }
    if (whole) {
      const float o = ll == 0.0f ? 0.0f : a / ll * sv;
      out[((int64_t)b * g.n_q_heads + hq0 + j) * D + d] = (uint16_t)(pack_bf16(o, 0.0f) & 0xFFFFu);
    } else {
      float *pp = part + ((int64_t)(hq0 + j) * ((int64_t)g.n_run + g.n_seqs) + x + b) * (2 + D);
      pp[2 + d] = a;
      if (d == 0) {
        pp[0] = M;
        pp[1] = ll;
      }
    }
  }
}

// Zero rows of sequence b (a block that takes whole sequences meets an empty one).
__device__ __forceinline__ void att_zero_rows(const AttnGeom &g, uint16_t *out, int G, int hq0, int b, int D) {
  for (int i = threadIdx.x; i < G * D; i += ATT_THREADS) out[((int64_t)b * g.n_q_heads + hq0) * D + i] = 0;
}

// Across 16-lane rows: the sum over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float att_xrow_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// The first run that holds a part of sequence b, and how many do.
__device__ __forceinline__ void att_live(const AttnGeom &g, const int32_t *seq_lens, void *table, int b, int32_t &x0,
                                         int32_t &n_live) {
  x0 = n_live = 0;
  if (g.n_seqs <= 64) {
    const int lane = threadIdx.x & 63;
    const AttnLanes l(g, lane < g.n_seqs ? seq_lens[lane] : 0);
    const uint32_t nb = __builtin_amdgcn_readlane(l.n, b);
    if (l.whole) {
      n_live = nb != 0;
    } else if (nb) {
      const uint32_t last = __builtin_amdgcn_readlane(l.incl, b) - 1;
      x0 = (int32_t)l.deal.run_of(last + 1 - nb);
      n_live = (int32_t)l.deal.run_of(last) - x0 + 1;
    }
  } else {
    const AttnTable t(table, g.n_seqs);
    x0 = t.x0[b];
    n_live = t.n_live[b];
  }
}

// Channel d of a row from its n parts (m, l, acc[D]), `step` floats apart, as bf16 times sv.  A
// wave owns 64 channels; its lanes hold the maxima and sums of 64 parts at a time, whose weights
// reach the channels by readlane, so there is no LDS and no barrier, and several parts' values
// are loaded before the first is used (1 x 2,048 positions, both passes: 20.4 -> 9.5 us, this
// one's share 4.0 -> 3.0; before, a block-wide table and one load at a time).
constexpr int CB_U = 8;  // parts whose values are loaded together
__device__ __forceinline__ uint16_t att_combine_row(const float *pp, int64_t step, int n, int d, float sv) {
  const int lane = threadIdx.x & 63;
  float M = -INFINITY, L = 0.0f, A = 0.0f;
  for (int base = 0; base < n; base += 64) {
    const int cnt = min(64, n - base);
    const float *p0 = pp + (int64_t)base * step;
    const float ms = lane < cnt ? p0[lane * step] : -INFINITY;
    const float ls = lane < cnt ? p0[lane * step + 1] : 0.0f;
    float v[CB_U];
#pragma unroll
    for (int u = 0; u < CB_U; ++u) v[u] = p0[min(u, cnt - 1) * step + 2 + d];
    const float Mn = fmaxf(M, xrow_max(row16_max(ms)));
    const float alpha = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
    const float w = Mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - Mn);
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
  // no positions (L = 0): zero
  return (uint16_t)(pack_bf16(L == 0.0f ? 0.0f : A / L * sv, 0.0f) & 0xFFFFu);
}

// ------------------------------------------------------------------ host side

// Blocks per group of query heads, and how the sequences are dealt to them.
struct AttnRuns {
  bool whole;
  int32_t unit;
  uint32_t tail, part, more;
  int64_t n_run, n_blk;
};
// When a kernel takes whole sequences (att_take_whole): with fewer sequences than runs, and with
// as many or more, where most runs would start anew anyway.
struct AttnSlack {
  uint32_t part_few, tail_few, part_many, tail_many, more;
};
// resident: blocks that the chip holds at once, one equal run each.  A number of groups that
// leaves a part of the CUs without a run takes up to four rounds of shorter ones where those
// fill the chip by 5% more (152 groups: 3 runs on 456 of 512, or 10 in three rounds: 16 x
// 1k-8k, 19 heads per kv head, D = 128 371 -> 311 us, D = 64 221 -> 164).
inline AttnRuns att_runs(int32_t n_seqs, int64_t groups, int64_t resident, int32_t unit, int32_t max_blocks,
                         int32_t page_size, const AttnSlack &slack) {
  AttnRuns p;
  p.unit = unit;
  // units of the longest sequence there can be (lengths are int32)
  const int64_t seq_units = ceil_div(std::min((int64_t)max_blocks * page_size, (int64_t)INT32_MAX), p.unit);
  int64_t slots = std::max<int64_t>(1, resident / groups);
  double per_round = (double)slots;
  for (int64_t rounds = 2; rounds <= 4; ++rounds) {
    const int64_t n = rounds * resident / groups;
    if ((double)n / rounds > 1.05 * per_round) {
      slots = n;
      per_round = (double)n / rounds;
    }
  }
  p.n_run = std::min(seq_units * n_seqs, slots);
  p.tail = n_seqs >= p.n_run ? slack.tail_many : slack.tail_few;
  p.part = n_seqs >= p.n_run ? slack.part_many : slack.part_few;
  p.more = slack.more;
  // Whole sequences whatever their lengths, without the merge's launch: one unit each, or at
  // most 512 positions where they fill half the chip (32 x 100-500: 10.2 us, in runs 17), or
  // so short that att_take_whole() says so anyway (128 x 100-600, 12 heads, D = 64: 26 -> 19).
  p.whole = seq_units == 1 || (seq_units * p.unit <= 512 && n_seqs >= slots / 2) ||
            seq_units <= p.tail;
  p.n_blk = p.whole ? n_seqs : std::max<int64_t>(p.n_run, n_seqs);  // room for either way of dealing
  return p;
}

// Partials, then the table (read by 8 bytes: 2 + head_dim is even).
inline size_t att_workspace_bytes(const AttnRuns &p, int32_t n_seqs, int32_t n_q_heads, int32_t head_dim) {
  return (size_t)(n_q_heads * (p.n_run + n_seqs) * (2 + head_dim)) * sizeof(float) +
         (n_seqs > 64 ? AttnTable::bytes(n_seqs, p.n_run) : 0);
}

// (g.group and g.n_group are the caller's)
inline AttnGeom att_geom(const AttnRuns &p, int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                         int32_t max_blocks, int32_t page_size, int64_t n_pages, float sm_scale) {
  AttnGeom g;
  g.n_q_heads = n_q_heads;
  g.n_kv_heads = n_kv_heads;
  g.head_dim = head_dim;
  g.page_size = page_size;
  g.max_blocks = max_blocks;
  g.n_seqs = n_seqs;
  g.n_run = (int32_t)p.n_run;
  g.tail = p.tail;
  g.part = p.part;
  g.more = p.more;
  g.unit = (uint32_t)p.unit;
  g.cap = (uint32_t)std::min((int64_t)max_blocks * page_size, (int64_t)INT32_MAX);
  g.whole = p.whole ? 1 : 0;
  g.group = g.n_group = 0;
  g.n_pages = n_pages;
  g.sm_scale = sm_scale;
  {  // magic division by the page size for positions below 2^31
    int sh = 0;
    while ((1LL << sh) < page_size) ++sh;
    g.p_shift = sh;
    g.p_magic = (uint32_t)(((1ULL << (31 + sh)) + (uint64_t)page_size - 1) / (uint64_t)page_size);
  }
  return g;
}

// The table of a call of more than 64 sequences that is dealt in runs (otherwise nothing).
int att_make_table(const AttnGeom &g, const int32_t *seq_lens, void *table, hipStream_t st);
// Pass 2: merges the partials of sequences that were cut; scales NULL stands for ones.
int att_combine(const float *part, const AttnGeom &g, const float *scales, const int32_t *seq_lens, uint16_t *out,
                void *table, hipStream_t st);

}  // namespace zx
