// zx_cross.hip -- attention of packed query rows to packed states of other lengths (cross attention
// to an encoder's states), and its gradients.  bf16 and fp16.
//
//   s_rt = sm_scale q_r . k_t,  p = softmax over the sequence's keys,  o_r = sum_t p_rt v_t,
//   lse_r = log2 sum_t 2^(s_rt log2 e);
//   with D_r = sum_d dO_rd o_rd:  p = 2^(s log2 e - lse),  dS = p (dO . v - D),
//   dq = sm_scale dS k,  dk = sm_scale dS^T q,  dv = p^T dO  (dk, dv over the KV head's query heads).
//
// All on v_mfma_f32_32x32x16, transposed so that the products' outputs are the next ones' operands
// (zx_attn_tile.h):
//   forward, dq:  columns are (query row, head of the KV head's group); K and V tiles of 64 keys in
//                 LDS; S^T = K Q^T, dP^T = V dO^T, O^T += V^T P^T, dQ^T += K^T dS^T
//   dk, dv:       columns are keys, their K in registers and their V's rows in LDS; Q and dO tiles
//                 of 32 (row, head) in LDS; S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// Every sum has a fixed order: gradients do not change from call to call (dq has a kernel of its
// own, two of seven products more than atomics would need).  Bound by the matrix products and
// the LDS reads that feed them; a call of few rows by the reads of K and V, its keys cut among
// blocks and the parts merged.
#include <algorithm>

#include "zx_attn_tile.h"
#include "zx_internal.h"

namespace zx {

// Rows [n][heads][D], strides in elements.
struct CrIn {
  const uint16_t *p;
  int64_t row, head;
};
constexpr int32_t CR_BY_KEYS = 1, CR_BY_ROWS = 2;
struct CrossArgs {
  CrIn q, k, v, o, g;       // g: the output's gradient
  const int32_t *cu_q, *cu_k, *k_lens;
  uint16_t *out;            // forward: out; dq
  uint16_t *dk, *dv;
  float *lse, *delta;       // [n_q_heads][n_q]
  float *part;              // forward: [split][n_q][n_q_heads][2 + D]; gradients: [split][rows][heads][D] each
  int32_t *err;
  int64_t n_q, n_k;
  int32_t n_q_heads, n_kv_heads, n_seqs, group;
  int32_t max_q, max_k;
  int32_t n_tile, n_split;  // tiles of a sequence and KV head at most, parts of each
  int32_t n_rest;           // blocks behind the others that clear the rows in no sequence
  uint32_t g_magic;         // c / group = (c * g_magic) >> (31 + g_shift) for c < 2^31
  int32_t g_shift;
  int32_t order;            // CR_BY_KEYS, CR_BY_ROWS: the sequences with the longest blocks first; 0: as they come
  float sm_scale;
};

// The row and the head within its group of pair c.
__device__ __forceinline__ uint32_t cr_pair(const CrossArgs &a, uint32_t c, uint32_t &head) {
  const uint32_t r = (uint32_t)(((uint64_t)c * a.g_magic) >> (31 + a.g_shift));
  head = c - r * (uint32_t)a.group;
  return r;
}

// Rows of the packed n that sequence b has: [lo, end), none outside, of which [lo, lo + n) are computed (at
// most `most`, and none of a sequence that begins before the first row).
struct CrSpan {
  int64_t lo, end;
  int32_t n;
};
__device__ __forceinline__ CrSpan cr_span(const int32_t *cu, int32_t b, int64_t n, int32_t most, int32_t &e) {
  const int64_t lo = cu[b], hi = cu[b + 1];
  if (lo < 0 || hi > n || hi - lo > most || hi < lo) e |= ZX_KERR_POS_RANGE;
  const int64_t from = max(lo, (int64_t)0), end = max(from, min(hi, n));
  return CrSpan{from, end, lo < 0 ? 0 : (int32_t)min(end - from, (int64_t)most)};
}
__device__ __forceinline__ int32_t cr_keys(const CrossArgs &a, int32_t b, int32_t n) {
  return a.k_lens ? max(0, min(a.k_lens[b], n)) : n;
}

// What a block does: tiles of one sequence and KV head on the same XCD (block ids go round the
// eight), so that what they read in common is in its L2; where blocks are long (cr_order) the
// sequences with the longest blocks first: the chip is left with short ones at the end (8 x 200-1,000 rows
// on 1,000-8,000 keys, 32/8 heads, D = 128: 350 -> 316 us, against those with the most pairs first; dk
// and dv of 4 x 1,000-2,048 rows on 2,000-8,192 gain 30 of 1,200).
struct CrItem {
  int32_t b, h, tile, split;
  bool any;
};
__device__ __forceinline__ CrItem cr_item(const CrossArgs &a) {
  const uint32_t xcd = blockIdx.x & 7u, i = blockIdx.x >> 3, per = (uint32_t)(a.n_tile * a.n_split);
  const uint32_t pair = (i / per) * 8 + xcd, rem = i - (i / per) * per;
  CrItem it;
  it.any = pair < (uint32_t)(a.n_seqs * a.n_kv_heads);
  it.b = (int32_t)(pair / (uint32_t)a.n_kv_heads);
  it.h = (int32_t)(pair - (uint32_t)it.b * (uint32_t)a.n_kv_heads);
  it.tile = (int32_t)(rem / (uint32_t)a.n_split);
  it.split = (int32_t)(rem - (uint32_t)it.tile * (uint32_t)a.n_split);
  if (a.order) {
    const int lane = threadIdx.x & 63;
    float w = -1.0f;
    if (lane < a.n_seqs) {
      const int32_t keys = a.cu_k[lane + 1] - a.cu_k[lane];
      w = (float)(a.order == CR_BY_ROWS ? a.cu_q[lane + 1] - a.cu_q[lane] : a.k_lens ? min(a.k_lens[lane], keys) : keys);
    }
    int before = lane < a.n_seqs ? 0 : 64;
    for (int s = 0; s < a.n_seqs; ++s) {
      const float other = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s));
      before += other > w || (other == w && s < lane);
    }
    it.b = __ffsll((long long)__ballot(before == it.b)) - 1;
    it.any &= it.b >= 0;
  }
  return it;
}
static unsigned cr_grid(const CrossArgs &a) {
  return (unsigned)(8 * ceil_div((int64_t)a.n_seqs * a.n_kv_heads, 8) * a.n_tile * a.n_split) + (unsigned)a.n_rest;
}

// The tile's loads, in registers until the LDS buffer is free.  Rows from n on are zeros (and not read).
template <int D, int R = CR_TILE> struct CrStage {
  static constexpr int LOADS = CrLds<D, R>::LOADS;
  uint4 x[LOADS];
  static __device__ __forceinline__ int row(int j) {
    return (int)threadIdx.x / CrLds<D>::CHUNKS + j * (CR_THREADS / CrLds<D>::CHUNKS);
  }
  static __device__ __forceinline__ int chunk() { return (int)threadIdx.x % CrLds<D>::CHUNKS; }
  // n >= 1 rows of `step` elements from p on (uniform; a tile's offsets fit 32 bits: cr_check_rows)
  __device__ __forceinline__ void load(const uint16_t *p, uint32_t step, int n) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      x[j] = *reinterpret_cast<const uint4 *>(p + ((uint32_t)min(row(j), n - 1) * step + 8u * (uint32_t)chunk()));
  }
  __device__ __forceinline__ void store(uint8_t *t, int n) const {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const uint4 z = row(j) < n ? x[j] : make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4 *>(cr_at<D>(t, row(j), 16 * chunk())) = z;
    }
  }
};

// Tiles [t_begin, t_end) in steps of `step` through two LDS buffers: load(t) issues a tile's loads (the
// first one's are under way, before the block reads its columns: 8 x 4,096 rows on 77 keys 29.6 -> 27.6
// us), store(buffer, t) writes them to LDS, compute(buffer, t) works on it.  (Loads two tiles ahead at
// D = 64 took the same time, or 4% more where they cost registers.)
template <class Load, class Store, class Compute>
__device__ __forceinline__ void cr_pipeline(int t_begin, int t_end, int step, Load load, Store store, Compute compute) {
  if (t_begin >= t_end) return;
  store(0, t_begin);
  __syncthreads();
  int buf = 0;
  for (int t = t_begin; t < t_end; t += step, buf ^= 1) {
    if (t + step < t_end) load(t + step);
    compute(buf, t);
    if (t + step < t_end) store(buf ^ 1, t + step);
    __syncthreads();
  }
}

// Columns of a wave: 32 CT of the block's 128 CT.
template <int D, int CT> struct CrCols {
  int32_t row[CT], head[CT];
  bool live[CT];
  __device__ __forceinline__ CrCols(const CrossArgs &a, int c0, int n_cols, int h, int64_t lo) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = c0 + 32 * (CT * wave + ct) + (lane & 31);
      live[ct] = c < n_cols;
      uint32_t hh;
      row[ct] = (int32_t)(lo + cr_pair(a, (uint32_t)min(c, n_cols - 1), hh));
      head[ct] = h * a.group + (int32_t)hh;
    }
  }
  // Their D channels as B operands (columns that are not there as zeros).
  __device__ __forceinline__ void load(const CrIn &x, att_u32x4 (&f)[CT][D / 16]) const {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const uint16_t *p = x.p + row[ct] * x.row + head[ct] * x.head + 8 * half;
#pragma unroll
      for (int kc = 0; kc < D / 16; ++kc) {
        const att_u32x4 w = *reinterpret_cast<const att_u32x4 *>(p + 16 * kc);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[ct][kc][i] = live[ct] ? w[i] : 0u;
      }
    }
  }
};

// Rows in no sequence (before the first, behind the last): zeros.  How many there are only the device
// knows: CR_REST blocks behind the others share them.
constexpr unsigned CR_REST = 64;
__device__ __forceinline__ bool cr_is_rest(const CrossArgs &a) { return blockIdx.x + (uint32_t)a.n_rest >= gridDim.x; }
__device__ __forceinline__ void cr_zero_rest(const CrossArgs &a, uint16_t *out, const int32_t *cu, int64_t n, int64_t width) {
  const int64_t lo = max((int64_t)0, min((int64_t)cu[0], n)), hi = max(lo, min((int64_t)cu[a.n_seqs], n));
  uint4 *p = reinterpret_cast<uint4 *>(out);
  const int64_t w = width / 8, step = (int64_t)a.n_rest * CR_THREADS;
  const int64_t first = (int64_t)(gridDim.x - 1 - blockIdx.x) * CR_THREADS + threadIdx.x;
  for (int64_t i = first; i < lo * w; i += step) p[i] = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t i = hi * w + first; i < n * w; i += step) p[i] = make_uint4(0u, 0u, 0u, 0u);
}

// Rows of a sequence that are not computed: zeros, by the first block of the sequence and KV head (`at`: its first
// element of a row, `width` elements).
__device__ __forceinline__ void cr_zero_behind(const CrItem &it, const CrSpan &s, uint16_t *out, int64_t row, int64_t at,
                                               int32_t width) {
  if (it.tile != 0 || it.split != 0 || s.lo + s.n >= s.end) return;  // uniform
  const int32_t w = width / 8;
  out += (s.lo + s.n) * row + at;
  for (int64_t i = threadIdx.x; i < (s.end - s.lo - s.n) * w; i += CR_THREADS)
    *reinterpret_cast<uint4 *>(out + i / w * row + 8 * (i % w)) = make_uint4(0u, 0u, 0u, 0u);
}

// ------------------------------------------------------------------ forward

template <class T, int D, int CT>
__global__ void __launch_bounds__(CR_THREADS, 2) cross_forward_kernel(CrossArgs a) {
  constexpr int KC = D / 16, DT = D / 32;
  __shared__ __attribute__((aligned(256))) uint8_t lds[2][2][CrLds<D>::BYTES];
  if (cr_is_rest(a)) {
    cr_zero_rest(a, a.out, a.cu_q, a.n_q, (int64_t)a.n_q_heads * D);
    return;
  }
  const CrItem it = cr_item(a);
  if (!it.any) return;
  int32_t e = 0;
  const CrSpan qs = cr_span(a.cu_q, it.b, a.n_q, a.max_q, e), ks = cr_span(a.cu_k, it.b, a.n_k, a.max_k, e);
  if (e && a.err && threadIdx.x == 0) atomicOr(a.err, e);
  if (a.n_rest) cr_zero_behind(it, qs, a.out, (int64_t)a.n_q_heads * D, (int64_t)it.h * a.group * D, a.group * D);
  const int n_cols = qs.n * a.group, c0 = it.tile * 32 * CT * CR_WAVES;
  if (c0 >= n_cols) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int keys = cr_keys(a, it.b, ks.n), units = (keys + CR_TILE - 1) / CR_TILE;
  const int t_begin = (int)((int64_t)units * it.split / a.n_split) * CR_TILE;
  const int t_end = min(keys, (int)((int64_t)units * (it.split + 1) / a.n_split) * CR_TILE);
  const uint16_t *kp = a.k.p + ks.lo * a.k.row + it.h * a.k.head, *vp = a.v.p + ks.lo * a.v.row + it.h * a.v.head;
  CrStage<D> sk, sv;
  auto load = [&](int t) {
    sk.load(kp + t * a.k.row, (uint32_t)a.k.row, min(CR_TILE, t_end - t));
    sv.load(vp + t * a.v.row, (uint32_t)a.v.row, min(CR_TILE, t_end - t));
  };
  if (t_begin < t_end) load(t_begin);
  const CrCols<D, CT> cols(a, c0, n_cols, it.h, qs.lo);
  const bool work = c0 + 32 * CT * wave < n_cols;  // uniform in the wave
  att_u32x4 q[CT][KC];
  cols.load(a.q, q);
  cr_f32x16 o[CT][DT];
  float m[CT], top[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[ct][dt] = cr_zero();
    m[ct] = top[ct] = CR_NONE;
    l[ct] = 0.0f;
  }
  // the scores' factor as a positive number: a negative one turns q's signs, 0 makes q zero
  const float scale = a.sm_scale * ATT_LOG2E, f = scale == 0.0f ? 1.0f : fabsf(scale);
  if (scale <= 0.0f) {
    const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u, keep = scale < 0.0f ? 0xFFFFFFFFu : 0u;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int kc = 0; kc < KC; ++kc)
#pragma unroll
        for (int i = 0; i < 4; ++i) q[ct][kc][i] = (q[ct][kc][i] ^ flip) & keep;
  }
  auto store = [&](int buf, int t) {
    sk.store(lds[buf][0], min(CR_TILE, t_end - t));
    sv.store(lds[buf][1], min(CR_TILE, t_end - t));
  };
  auto compute = [&](int buf, int t) {
    if (work) {
      uint8_t *lk = lds[buf][0], *lv = lds[buf][1];
      cr_f32x16 s[CT][2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) s[ct][kt] = cr_zero();
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          const att_u32x4 k = cr_rows<D>(lk, kt, kc, lane);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) s[ct][kt] = T::mfma(k, q[ct][kc], s[ct][kt]);
        }
      }
      if (t + CR_TILE > t_end) {  // uniform
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (t + 32 * kt + cr_row(i, lane) >= t_end) s[ct][kt][i] = -INFINITY;
      }
      float mx[CT];
      bool grew = false;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        mx[ct] = s[ct][0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i) mx[ct] = __builtin_elementwise_maximum(mx[ct], s[ct][i / 16][i % 16]);
        grew |= mx[ct] > top[ct];
      }
      if (__builtin_amdgcn_ballot_w64(grew)) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const float m_new = fmaxf(m[ct], cr_halves_max(mx[ct]) * f - T::BIAS);
          const float alpha = __builtin_amdgcn_exp2f(m[ct] - m_new);
          m[ct] = m_new;
          top[ct] = (m_new + (CR_LAZY + T::BIAS)) / f;
          l[ct] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[ct][dt][i] *= alpha;
        }
      }
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        att_u32x4 p[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][kt][i], f, -m[ct]));
            l[ct] += x[i];
          }
          cr_operands<T>(x, p[ct]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const att_u32x4 v = cr_cols<D>(lv, 2 * kt + c, dt, lane);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) o[ct][dt] = T::mfma(v, p[ct][c], o[ct][dt]);
          }
      }
    }
  };
  cr_pipeline(t_begin, t_end, CR_TILE, load, store, compute);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (!cols.live[ct]) continue;
    const float sum = cr_halves_sum(l[ct]);
    const int64_t at = (int64_t)cols.row[ct] * a.n_q_heads + cols.head[ct];
    if (a.n_split == 1) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint16_t *row = a.out + at * D + 4 * (lane >> 5);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<uint2 *>(row + 32 * dt + 2 * i) =
              sum == 0.0f ? make_uint2(0u, 0u)
                          : make_uint2(T::pack(o[ct][dt][i] * inv, o[ct][dt][i + 1] * inv),
                                       T::pack(o[ct][dt][i + 2] * inv, o[ct][dt][i + 3] * inv));
      if (a.lse && lane < 32)
        a.lse[(int64_t)cols.head[ct] * a.n_q + cols.row[ct]] = sum == 0.0f ? -INFINITY : m[ct] + __builtin_amdgcn_logf(sum);
    } else {
      float *pp = a.part + ((int64_t)it.split * a.n_q * a.n_q_heads + at) * (2 + D);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 2)
          *reinterpret_cast<float2 *>(pp + 2 + 32 * dt + cr_row(i, lane)) = make_float2(o[ct][dt][i], o[ct][dt][i + 1]);
      if (lane < 32) *reinterpret_cast<float2 *>(pp) = make_float2(m[ct], sum);
    }
  }
}

// The sequence that computes a packed row, or -1: none, or the row is beyond what is computed of it (cr_span).
__device__ __forceinline__ int32_t cr_seq_of(const int32_t *cu, int32_t n_seqs, int64_t row, int32_t most) {
  int32_t lo = 0, hi = n_seqs - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return cu[lo] >= 0 && row >= cu[lo] && row < cu[lo + 1] && row - cu[lo] < most ? lo : -1;
}

// Rows whose keys were cut: D threads per (row, head).
template <class T, int D> __global__ void __launch_bounds__(256) cross_merge_kernel(CrossArgs a) {
  const int64_t at = (int64_t)blockIdx.x * (256 / D) + threadIdx.x / D, row = at / a.n_q_heads;
  if (row >= a.n_q) return;
  if (cr_seq_of(a.cu_q, a.n_seqs, row, a.max_q) < 0) return;
  const int d = threadIdx.x % D;
  const int64_t step = a.n_q * a.n_q_heads * (2 + D);
  const float *pp = a.part + at * (2 + D);
  float M = CR_NONE, L = 0.0f, A = 0.0f;
  for (int s0 = 0; s0 < a.n_split; s0 += 8) {
    float2 ml[8];
    float v[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float *p = pp + min(s0 + s, a.n_split - 1) * step;
      ml[s] = *reinterpret_cast<const float2 *>(p);
      v[s] = p[2 + d];
    }
    float Mn = M;
#pragma unroll
    for (int s = 0; s < 8; ++s) Mn = fmaxf(Mn, ml[s].x);
    const float alpha = __builtin_amdgcn_exp2f(M - Mn);
    L *= alpha;
    A *= alpha;
    M = Mn;
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s0 + s < a.n_split) {
        const float w = __builtin_amdgcn_exp2f(ml[s].x - M);
        L += w * ml[s].y;
        A += w * v[s];
      }
  }
  a.out[at * D + d] = (uint16_t)(T::pack(L == 0.0f ? 0.0f : A / L, 0.0f) & 0xFFFFu);
  if (a.lse && d == 0)
    a.lse[(at - row * a.n_q_heads) * a.n_q + row] = L == 0.0f ? -INFINITY : M + __builtin_amdgcn_logf(L);
}

// ------------------------------------------------------------------ gradients

// dS is one of the two 16-bit operands of dq's and dk's products, and in fp16 its size matters: on 1,500 keys,
// with output gradients of 1e-4, it lies near 2^-21, where fp16 has 3 bits.  So in fp16 it is carried
// times a power of two that every column (dq: a row, dk: a key) finds for itself and lowers when a value
// exceeds 2^15, to where the largest is in [2^7, 2^8); what was summed before is rescaled, the sum divided at
// the end.  So values keep fp16's 11 bits whatever the gradient's size, small ones are off by 2^-32 of the
// largest so far at most, and none overflows.  (D = 64, 256 rows on 1,500 and 8,000 keys, gradients of 1e-4: dq
// 1.9e-2 and 1.0e-1 off without it, 3.9e-3 and 9.3e-3 with it, which is its own last rounding; gradients of
// 16 x 50-448 rows on 1,500 keys, 12 heads, 128 -> 133 us, of long ones at D = 128 1,973 -> 1,998.  bf16, with
// fp32's exponents, needs none of it.)
constexpr float CR_DS_FIRST = 0x1p64f;  // |dP| < 2^38 at D = 64 (128: 2^39): no overflow in fp32
constexpr float CR_DS_MOST = 0x1p15f;
template <class T> constexpr bool CR_SCALED = T::BIAS != 0.0f;

// The factor by which a column whose largest of these values (over both of its lanes) is w goes down.
__device__ __forceinline__ float cr_lower(float w) {
  // (2^(e-1) <= w < 2^e; of an infinity e is 0)
  return w > CR_DS_MOST ? __builtin_amdgcn_ldexpf(1.0f, min(8 - __builtin_amdgcn_frexp_expf(w), 0)) : 1.0f;
}
// Lowers a column's factor, with what x and `sums` have of it, where x needs that.
template <int DT> __device__ __forceinline__ void cr_fit(float (&x)[16], float &up, cr_f32x16 (&sums)[DT]) {
  float mx = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, fabsf(x[i]));
  if (__builtin_amdgcn_ballot_w64(mx > CR_DS_MOST)) {
    const float a = cr_lower(cr_halves_max(mx));
    up *= a;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= a;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[dt][i] *= a;
  }
}

// dq, and on the way D_r for the other kernel.
template <class T, int D>
__global__ void __launch_bounds__(CR_THREADS, D == 64 ? 3 : 2) cross_dq_kernel(CrossArgs a) {
  constexpr int CT = 1, KC = D / 16, DT = D / 32;
  __shared__ __attribute__((aligned(256))) uint8_t lds[2][2][CrLds<D>::BYTES];
  if (cr_is_rest(a)) {
    cr_zero_rest(a, a.out, a.cu_q, a.n_q, (int64_t)a.n_q_heads * D);
    return;
  }
  const CrItem it = cr_item(a);
  if (!it.any) return;
  int32_t e = 0;
  const CrSpan qs = cr_span(a.cu_q, it.b, a.n_q, a.max_q, e), ks = cr_span(a.cu_k, it.b, a.n_k, a.max_k, e);
  if (e && a.err && threadIdx.x == 0) atomicOr(a.err, e);
  cr_zero_behind(it, qs, a.out, (int64_t)a.n_q_heads * D, (int64_t)it.h * a.group * D, a.group * D);
  const int n_cols = qs.n * a.group, c0 = it.tile * 32 * CT * CR_WAVES;
  if (c0 >= n_cols) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int keys = cr_keys(a, it.b, ks.n), units = (keys + CR_TILE - 1) / CR_TILE;
  const int t_begin = (int)((int64_t)units * it.split / a.n_split) * CR_TILE;
  const int t_end = min(keys, (int)((int64_t)units * (it.split + 1) / a.n_split) * CR_TILE);
  const uint16_t *kp = a.k.p + ks.lo * a.k.row + it.h * a.k.head, *vp = a.v.p + ks.lo * a.v.row + it.h * a.v.head;
  CrStage<D> sk, sv;
  auto load = [&](int t) {
    sk.load(kp + t * a.k.row, (uint32_t)a.k.row, min(CR_TILE, t_end - t));
    sv.load(vp + t * a.v.row, (uint32_t)a.v.row, min(CR_TILE, t_end - t));
  };
  constexpr bool EARLY = D == 64;  // (at D = 128 ten registers would be spilled)
  if (EARLY && t_begin < t_end) load(t_begin);
  const CrCols<D, CT> cols(a, c0, n_cols, it.h, qs.lo);
  const bool work = c0 + 32 * CT * wave < n_cols;
  att_u32x4 q[CT][KC], g[CT][KC];
  cols.load(a.q, q);
  cols.load(a.g, g);
  float lse[CT], delta[CT], up[CT];
  cr_f32x16 dq[CT][DT];
  const bool few = a.n_split == 1 && keys <= 2 * CR_TILE;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int64_t at = (int64_t)cols.head[ct] * a.n_q + cols.row[ct];
    lse[ct] = a.lse[at];
    up[ct] = CR_SCALED<T> ? CR_DS_FIRST : 1.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dq[ct][dt] = cr_zero();
    if (few) continue;
    const uint16_t *p = a.o.p + cols.row[ct] * a.o.row + cols.head[ct] * a.o.head + 8 * (lane >> 5);
    float sum = 0.0f;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const att_u32x4 w = *reinterpret_cast<const att_u32x4 *>(p + 16 * kc);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum = __builtin_fmaf(T::lo(w[i]), T::lo(g[ct][kc][i]), sum);
        sum = __builtin_fmaf(T::hi(w[i]), T::hi(g[ct][kc][i]), sum);
      }
    }
    delta[ct] = cr_halves_sum(sum);
    if (it.split == 0 && cols.live[ct] && lane < 32) a.delta[at] = delta[ct];
  }
  const float scale = a.sm_scale * ATT_LOG2E;
  auto store = [&](int buf, int t) {
    sk.store(lds[buf][0], min(CR_TILE, t_end - t));
    sv.store(lds[buf][1], min(CR_TILE, t_end - t));
  };
  auto products = [&](int buf, int kt, cr_f32x16 (&s)[CT], cr_f32x16 (&dp)[CT]) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) s[ct] = dp[ct] = cr_zero();
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const att_u32x4 k = cr_rows<D>(lds[buf][0], kt, kc, lane), v = cr_rows<D>(lds[buf][1], kt, kc, lane);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        s[ct] = T::mfma(k, q[ct][kc], s[ct]);
        dp[ct] = T::mfma(v, g[ct][kc], dp[ct]);
      }
    }
  };
  auto compute = [&](int buf, int t) {
    if (work) {
      uint8_t *lk = lds[buf][0];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        cr_f32x16 s[CT], dp[CT];
        products(buf, kt, s, dp);
        att_u32x4 ds[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][i], scale, -lse[ct]));
            x[i] = p * (CR_SCALED<T> ? __builtin_fmaf(dp[ct][i], up[ct], -delta[ct] * up[ct]) : dp[ct][i] - delta[ct]);
          }
          if (t + CR_TILE > t_end) {  // uniform
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (t + 32 * kt + cr_row(i, lane) >= t_end) x[i] = 0.0f;
          }
          if constexpr (CR_SCALED<T>) cr_fit(x, up[ct], dq[ct]);
          cr_operands<T>(x, ds[ct]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const att_u32x4 k = cr_cols<D>(lk, 2 * kt + c, dt, lane);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) dq[ct][dt] = T::mfma(k, ds[ct][c], dq[ct][dt]);
          }
      }
    }
  };
  if (few) {
    // All the keys fit the two buffers: D_r = sum_t p dP, which needs no rounded out.  (What out's last
    // rounding adds to dS weighs the more the fewer the keys: of dq's error at 6 keys a third.)
    for (int t = 0, buf = 0; t < t_end; t += CR_TILE, ++buf) {
      if (!EARLY || t) load(t);
      store(buf, t);
    }
    __syncthreads();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) delta[ct] = 0.0f;
    if (work) {
      for (int t = 0, buf = 0; t < t_end; t += CR_TILE, ++buf) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          cr_f32x16 s[CT], dp[CT];
          products(buf, kt, s, dp);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][i], scale, -lse[ct])) * dp[ct][i];
              delta[ct] += t + 32 * kt + cr_row(i, lane) < t_end ? x : 0.0f;
            }
        }
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      delta[ct] = cr_halves_sum(delta[ct]);
      if (cols.live[ct] && lane < 32) a.delta[(int64_t)cols.head[ct] * a.n_q + cols.row[ct]] = delta[ct];
    }
    for (int t = 0, buf = 0; t < t_end; t += CR_TILE, ++buf) compute(buf, t);
  } else {
    if (!EARLY && t_begin < t_end) load(t_begin);
    cr_pipeline(t_begin, t_end, CR_TILE, load, store, compute);
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (!cols.live[ct]) continue;
    const int64_t at = ((int64_t)cols.row[ct] * a.n_q_heads + cols.head[ct]) * D + 4 * (lane >> 5);
    const float down = a.sm_scale / up[ct];
    if (a.n_split == 1) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<uint2 *>(a.out + at + 32 * dt + 2 * i) =
              make_uint2(T::pack(dq[ct][dt][i] * down, dq[ct][dt][i + 1] * down),
                         T::pack(dq[ct][dt][i + 2] * down, dq[ct][dt][i + 3] * down));
    } else {
      float *pp = a.part + (int64_t)it.split * a.n_q * a.n_q_heads * D + at;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4 *>(pp + 32 * dt + 2 * i) =
              make_float4(dq[ct][dt][i] * down, dq[ct][dt][i + 1] * down, dq[ct][dt][i + 2] * down,
                          dq[ct][dt][i + 3] * down);
    }
  }
}

// dk and dv of 128 keys, a wave 32 of them.
template <class T, int D>
__global__ void __launch_bounds__(CR_THREADS, D == 64 ? 3 : 2) cross_dkv_kernel(CrossArgs a) {
  constexpr int R = 32;  // rows per tile
  constexpr int KC = D / 16, DT = D / 32;
  using VRows = CrRowsOnly<D>;
  __shared__ __attribute__((aligned(256))) uint8_t lv[32 * CR_WAVES * VRows::ROW];  // V's rows
  __shared__ __attribute__((aligned(256))) uint8_t lds[2][2][CrLds<D, R>::BYTES];
  __shared__ __attribute__((aligned(16))) float sm_lse[2][R], sm_delta[2][R];
  if (cr_is_rest(a)) {
    cr_zero_rest(a, a.dk, a.cu_k, a.n_k, (int64_t)a.n_kv_heads * D);
    cr_zero_rest(a, a.dv, a.cu_k, a.n_k, (int64_t)a.n_kv_heads * D);
    return;
  }
  const CrItem it = cr_item(a);
  if (!it.any) return;
  int32_t e = 0;  // (reported with dq)
  const CrSpan qs = cr_span(a.cu_q, it.b, a.n_q, a.max_q, e), ks = cr_span(a.cu_k, it.b, a.n_k, a.max_k, e);
  const int key0 = it.tile * 32 * CR_WAVES;
  cr_zero_behind(it, ks, a.dk, (int64_t)a.n_kv_heads * D, (int64_t)it.h * D, D);
  cr_zero_behind(it, ks, a.dv, (int64_t)a.n_kv_heads * D, (int64_t)it.h * D, D);
  if (key0 >= ks.n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int keys = cr_keys(a, it.b, ks.n);
  const int n_cols = key0 < keys ? qs.n * a.group : 0, units = (n_cols + R - 1) / R;
  const int t_begin = (int)((int64_t)units * it.split / a.n_split) * R;
  const int t_end = min(n_cols, (int)((int64_t)units * (it.split + 1) / a.n_split) * R);
  const int wk = key0 + 32 * wave;  // the wave's first key
  const bool work = wk < keys, live = wk + (lane & 31) < keys;
  att_u32x4 k[KC];
  cr_f32x16 dk[DT], dv[DT];
  {
    const int64_t row = ks.lo + max(0, min(wk + (lane & 31), keys - 1));
    const uint16_t *kp = a.k.p + row * a.k.row + it.h * a.k.head + 8 * (lane >> 5);
    // (keys that are not there are columns of their own: cleared where they are written)
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) k[kc] = *reinterpret_cast<const att_u32x4 *>(kp + 16 * kc);
  }
  uint8_t *const my_v = VRows::at(lv, 32 * wave + (lane & 31), 16 * (lane >> 5));
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dk[dt] = dv[dt] = cr_zero();
  const float scale = a.sm_scale * ATT_LOG2E;
  const uint16_t *qp = a.q.p + qs.lo * a.q.row + (int64_t)it.h * a.group * a.q.head;
  const uint16_t *gp = a.g.p + qs.lo * a.g.row + (int64_t)it.h * a.group * a.g.head;
  CrStage<D, R> sq, sg;
  float my_lse = 0.0f, my_delta = 0.0f;
  auto load = [&](int t) {
    const int n = min(R, t_end - t);
    uint32_t hh;
    const uint32_t r0 = cr_pair(a, (uint32_t)t, hh);  // uniform
    const uint16_t *q = qp + (int64_t)r0 * a.q.row, *g = gp + (int64_t)r0 * a.g.row;
#pragma unroll
    for (int j = 0; j < CrStage<D, R>::LOADS; ++j) {
      const uint32_t r = cr_pair(a, (uint32_t)(t + min(CrStage<D, R>::row(j), n - 1)), hh) - r0;
      const uint32_t c = 8u * (uint32_t)CrStage<D, R>::chunk();
      sq.x[j] = *reinterpret_cast<const uint4 *>(q + (r * (uint32_t)a.q.row + hh * (uint32_t)a.q.head + c));
      sg.x[j] = *reinterpret_cast<const uint4 *>(g + (r * (uint32_t)a.g.row + hh * (uint32_t)a.g.head + c));
    }
    if (threadIdx.x < R) {
      const uint32_t r = cr_pair(a, (uint32_t)(t + min((int)threadIdx.x, n - 1)), hh);
      const int64_t at = (int64_t)(it.h * a.group + (int32_t)hh) * a.n_q + qs.lo + r;
      my_lse = a.lse[at];
      my_delta = a.delta[at];
    }
  };
  if (t_begin < t_end) load(t_begin);
  {
    const uint16_t *vp = a.v.p + ks.lo * a.v.row + it.h * a.v.head;
    for (int i = threadIdx.x; i < 32 * CR_WAVES * D / 8; i += CR_THREADS) {
      const int r = i / (D / 8), c = i % (D / 8);
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (key0 + r < keys) w = *reinterpret_cast<const uint4 *>(vp + (key0 + r) * a.v.row + 8 * c);
      *reinterpret_cast<uint4 *>(VRows::at(lv, r, 16 * c)) = w;
    }
  }
  auto store = [&](int buf, int t) {
    const int n = min(R, t_end - t);
    sq.store(lds[buf][0], n);
    sg.store(lds[buf][1], n);
    if (threadIdx.x < R) {  // (a row that is not there: weights of 0)
      sm_lse[buf][threadIdx.x] = (int)threadIdx.x < n ? my_lse - T::BIAS : INFINITY;
      sm_delta[buf][threadIdx.x] = (int)threadIdx.x < n ? my_delta : 0.0f;
    }
  };
  const float unbias = __builtin_amdgcn_exp2f(-T::BIAS);
  float up = CR_SCALED<T> ? CR_DS_FIRST * unbias : unbias;  // of dS, from the weights as they are carried
  auto compute = [&](int buf, int) {
    if (!work) return;
    uint8_t *lq = lds[buf][0], *lg = lds[buf][1];
    cr_f32x16 s = cr_zero(), dp = cr_zero();
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      s = T::mfma(cr_rows<D>(lq, 0, kc, lane), k[kc], s);
      dp = T::mfma(cr_rows<D>(lg, 0, kc, lane), *reinterpret_cast<const att_u32x4 *>(my_v + 32 * kc), dp);
    }
    att_u32x4 p[2], ds[2];
    float x[16], y[16];
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int row = 8 * i4 + 4 * (lane >> 5);
      const att_f32x4 lse = *reinterpret_cast<const att_f32x4 *>(&sm_lse[buf][row]);
      const att_f32x4 delta = *reinterpret_cast<const att_f32x4 *>(&sm_delta[buf][row]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 4 * i4 + j;
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale, -lse[j]));
        y[i] = x[i] * up * (dp[i] - delta[j]);
      }
    }
    if constexpr (CR_SCALED<T>) cr_fit(y, up, dk);
    cr_operands<T>(x, p);
    cr_operands<T>(y, ds);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        dv[dt] = T::mfma(cr_cols<D>(lg, c, dt, lane), p[c], dv[dt]);
        dk[dt] = T::mfma(cr_cols<D>(lq, c, dt, lane), ds[c], dk[dt]);
      }
  };
  cr_pipeline(t_begin, t_end, R, load, store, compute);
  const float down = a.sm_scale * (unbias / up);
  const int key = wk + (lane & 31);
  if (key >= ks.n) return;
  const int64_t at = ((ks.lo + key) * a.n_kv_heads + it.h) * D + 4 * (lane >> 5), all = a.n_k * a.n_kv_heads * D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = live ? dk[dt][i + j] * down : 0.0f;
        y[j] = live ? dv[dt][i + j] * unbias : 0.0f;
      }
      const int64_t w = at + 32 * dt + 2 * i;
      if (a.n_split == 1) {
        *reinterpret_cast<uint2 *>(a.dk + w) = make_uint2(T::pack(x[0], x[1]), T::pack(x[2], x[3]));
        *reinterpret_cast<uint2 *>(a.dv + w) = make_uint2(T::pack(y[0], y[1]), T::pack(y[2], y[3]));
      } else {
        float *pp = a.part + 2 * (int64_t)it.split * all + w;
        *reinterpret_cast<float4 *>(pp) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(pp + all) = make_float4(y[0], y[1], y[2], y[3]);
      }
    }
}

// Sums of the parts of a gradient, in order: [n_split] parts `step` floats apart, 8 values per thread;
// blocks of y = 1: of a second one, whose parts lie behind the first one's.
template <class T>
__global__ void __launch_bounds__(256) cross_sum_kernel(const float *part, int64_t step, int32_t n_split, uint16_t *out0,
                                                        uint16_t *out1, const int32_t *cu, int32_t n_seqs, int64_t n, int64_t width,
                                                        int32_t most) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= n * width) return;
  const int64_t row = at / width;
  if (cr_seq_of(cu, n_seqs, row, most) < 0) return;  // zeros already
  uint16_t *out = blockIdx.y ? out1 : out0;
  if (blockIdx.y) part += n * width;
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < n_split; ++s) {
    const att_f32x4 *p = reinterpret_cast<const att_f32x4 *>(part + s * step + at);
    const att_f32x4 u = p[0], v = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] += u[i];
      x[4 + i] += v[i];
    }
  }
  *reinterpret_cast<uint4 *>(out + at) =
      make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
}

}  // namespace zx

using namespace zx;

// How a kernel is cut: column (or key) tiles per wave, tiles of a pair of sequence and KV head,
// parts of a tile where the tiles do not fill the chip.
struct CrossPlan {
  int ct;
  int64_t n_tile, n_split;
};
// Ranking the sequences costs every block about 1 us per 64 of them: for blocks of 16 tiles and more.
static int32_t cr_order(int32_t n_seqs, int64_t length, int32_t by) {
  return n_seqs > 1 && n_seqs <= 64 && length >= 16 * CR_TILE ? by : 0;
}
static CrossPlan cr_plan(int64_t pairs, int64_t columns, int64_t length, int ct, int64_t per_cu, int64_t units_least) {
  CrossPlan p;
  p.ct = ct;
  p.n_tile = std::max<int64_t>(1, ceil_div(columns, 32 * ct * CR_WAVES));
  const int64_t blocks = pairs * p.n_tile, slots = per_cu * num_cus();
  const int64_t units = ceil_div(length, CR_TILE);
  p.n_split = std::max<int64_t>(1, std::min<int64_t>({slots / std::max<int64_t>(1, blocks), units / units_least, 64}));
  return p;
}
static CrossPlan cr_forward_plan(int32_t n_seqs, int32_t n_kv_heads, int32_t group, int32_t D, int32_t max_q, int32_t max_k) {
  const int64_t columns = (int64_t)max_q * group, pairs = (int64_t)n_seqs * n_kv_heads;
  // Two column tiles per wave halve the LDS reads of K and V per product, where they leave two
  // waves per SIMD (D = 64) and tiles enough: 4 x 2,048 rows x 4 heads on 4,096 keys 302 us against
  // 340; 16 x 448 rows on 1,500 keys, 12 heads 106 against 57.  (D = 128, one wave per SIMD then: 4 x
  // 2,048 rows, 32/8 heads, on 8,192 keys 1,364 against 1,202.)
  const int ct = D == 64 && columns >= 1024 && pairs * ceil_div(columns, 256) >= 4 * num_cus() ? 2 : 1;
  return cr_plan(pairs, columns, max_k, ct, D == 64 && ct == 1 ? 3 : 2, 2);
}
static CrossPlan cr_dq_plan(int32_t n_seqs, int32_t n_kv_heads, int32_t group, int32_t D, int32_t max_q, int32_t max_k) {
  return cr_plan((int64_t)n_seqs * n_kv_heads, (int64_t)max_q * group, max_k, 1, D == 64 ? 3 : 2, 4);
}
static CrossPlan cr_dkv_plan(int32_t n_seqs, int32_t n_kv_heads, int32_t group, int32_t D, int32_t max_q, int32_t max_k) {
  return cr_plan((int64_t)n_seqs * n_kv_heads, max_k, (int64_t)max_q * group, 1, D == 64 ? 3 : 2, 4);
}
static bool cr_dims_ok(int64_t n_q, int64_t n_k, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t n_seqs,
                       int32_t max_q, int32_t max_k) {
  return n_q >= 0 && n_k >= 0 && n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0 &&
         (head_dim == 64 || head_dim == 128) && n_seqs > 0 && max_q >= 0 && max_k >= 0;
}

static size_t cr_forward_bytes(const CrossPlan &p, int64_t n_q, int32_t n_q_heads, int32_t D) {
  return p.n_split > 1 ? (size_t)(p.n_split * n_q * n_q_heads * (2 + D)) * sizeof(float) : 0;
}
extern "C" size_t zx_cross_attention_workspace_bytes(int64_t n_q, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                     int32_t n_seqs, int32_t max_q_per_seq, int32_t max_k_per_seq) {
  if (!cr_dims_ok(n_q, 0, n_q_heads, n_kv_heads, head_dim, n_seqs, max_q_per_seq, max_k_per_seq)) return 0;
  return cr_forward_bytes(cr_forward_plan(n_seqs, n_kv_heads, n_q_heads / n_kv_heads, head_dim,
                                          (int32_t)std::min<int64_t>(max_q_per_seq, n_q), max_k_per_seq),
                          n_q, n_q_heads, head_dim);
}

struct CrossGradBytes {
  size_t delta, part;
};
static CrossGradBytes cr_grad_bytes(const CrossPlan &dq, const CrossPlan &dkv, int64_t n_q, int64_t n_k, int32_t n_q_heads,
                                    int32_t n_kv_heads, int32_t D) {
  const size_t a = dq.n_split > 1 ? (size_t)(dq.n_split * n_q * n_q_heads * D) * sizeof(float) : 0;
  const size_t b = dkv.n_split > 1 ? (size_t)(2 * dkv.n_split * n_k * n_kv_heads * D) * sizeof(float) : 0;
  return CrossGradBytes{align256((size_t)(n_q * n_q_heads) * sizeof(float)), std::max(a, b)};
}
extern "C" size_t zx_cross_attention_backward_workspace_bytes(int64_t n_q, int64_t n_k, int32_t n_q_heads,
                                                              int32_t n_kv_heads, int32_t head_dim, int32_t n_seqs,
                                                              int32_t max_q_per_seq, int32_t max_k_per_seq) {
  if (!cr_dims_ok(n_q, n_k, n_q_heads, n_kv_heads, head_dim, n_seqs, max_q_per_seq, max_k_per_seq)) return 0;
  const int32_t group = n_q_heads / n_kv_heads, mq = (int32_t)std::min<int64_t>(max_q_per_seq, n_q);
  const int32_t mk = (int32_t)std::min<int64_t>(max_k_per_seq, n_k);
  const CrossGradBytes b = cr_grad_bytes(cr_dq_plan(n_seqs, n_kv_heads, group, head_dim, mq, mk),
                                         cr_dkv_plan(n_seqs, n_kv_heads, group, head_dim, mq, mk), n_q, n_k, n_q_heads,
                                         n_kv_heads, head_dim);
  return b.delta + b.part;
}

static int cr_check(const char *what, int dtype, const CrossArgs &a, int32_t head_dim) {
  ZX_REQUIRE(dtype == ZX_BF16 || dtype == ZX_F16, "%s: dtype must be bf16 or f16", what);
  ZX_REQUIRE(a.n_q >= 0 && a.n_k >= 0 && a.n_q_heads > 0 && a.n_kv_heads > 0 && a.n_seqs > 0 && a.max_q >= 0 && a.max_k >= 0,
             "%s: sizes must be positive", what);
  ZX_REQUIRE(a.n_q_heads % a.n_kv_heads == 0, "%s: n_q_heads must be a multiple of n_kv_heads", what);
  if (head_dim != 64 && head_dim != 128)
    return fail(ZX_ERR_UNSUPPORTED, "%s: head_dim %d not in {64, 128}", what, head_dim);
  constexpr int64_t MOST = (1LL << 31) - 4096;  // rounded up to tiles they fit 31 bits
  if (a.n_q >= MOST || a.n_k >= MOST || a.n_q * a.n_q_heads >= MOST || a.n_k * a.n_kv_heads >= MOST)
    return fail(ZX_ERR_UNSUPPORTED, "%s: too many rows", what);
  return ZX_OK;
}
// Strided rows: channels contiguous, every head's row 16-byte aligned, a tile's offsets below 2^31 bytes.
static int cr_check_rows(const char *what, const char *name, const CrIn &x, int64_t group) {
  ZX_REQUIRE(x.p, "%s: null pointer", what);
  ZX_REQUIRE(aligned16(x.p) && x.row % 8 == 0 && x.head % 8 == 0 && x.row >= 0 && x.head >= 0,
             "%s: every row of a head of %s must be 16-byte aligned, with strides that are not negative", what, name);
  if (x.row >= (1LL << 23) || (group > 1 && x.head >= (1LL << 29) / group))
    return fail(ZX_ERR_UNSUPPORTED, "%s: strides of %s are too large", what, name);
  return ZX_OK;
}

// Whether any of `bytes` from `out` on lies between the first and the last element of n x heads rows of x.
static bool cr_meets(const void *out, int64_t bytes, const CrIn &x, int64_t n, int64_t heads, int64_t d) {
  if (!out || !x.p || bytes <= 0 || n <= 0) return false;
  typedef __int128 wide;  // (a stride is anything)
  const wide at = (wide) reinterpret_cast<uintptr_t>(x.p), o = (wide) reinterpret_cast<uintptr_t>(out);
  return o < at + 2 * ((n - 1) * (wide)x.row + (heads - 1) * (wide)x.head + d) && at < o + bytes;
}

static void cr_group(CrossArgs &a) {
  a.group = a.n_q_heads / a.n_kv_heads;
  int sh = 0;
  while ((1LL << sh) < a.group) ++sh;
  a.g_shift = sh;
  a.g_magic = (uint32_t)(((1ULL << (31 + sh)) + (uint64_t)a.group - 1) / (uint64_t)a.group);
}

template <class T, int D> static int cr_forward(CrossArgs a, const CrossPlan &p, hipStream_t st) {
  const unsigned grid = cr_grid(a);
  if (D == 64 && p.ct == 2) cross_forward_kernel<T, 64, 2><<<grid, CR_THREADS, 0, st>>>(a);
  else cross_forward_kernel<T, D, 1><<<grid, CR_THREADS, 0, st>>>(a);
  const int rc = check_launch("cross_forward");
  if (rc || a.n_split == 1) return rc;
  cross_merge_kernel<T, D><<<(unsigned)ceil_div(a.n_q * a.n_q_heads, 256 / D), 256, 0, st>>>(a);
  return check_launch("cross_merge");
}

extern "C" int zx_cross_attention(int dtype, const void *q, int64_t n_q, int64_t q_row, int64_t q_head, int32_t n_q_heads,
                                  const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row, int64_t v_head,
                                  int64_t n_k, int32_t n_kv_heads, int32_t head_dim, const int32_t *cu_q,
                                  const int32_t *cu_k, const int32_t *k_lens, int32_t n_seqs, int32_t max_q_per_seq,
                                  int32_t max_k_per_seq, float sm_scale, int32_t flags, void *out, float *lse2, int32_t *err,
                                  void *workspace, size_t workspace_bytes, zx_stream_t stream) {
  clear_error();
  ZX_REQUIRE(!(flags & ~ZX_CROSS_ZERO_REST), "cross_attention: unknown flag bits 0x%x", (unsigned)flags);
  CrossArgs a = {};
  a.q = {static_cast<const uint16_t *>(q), q_row, q_head};
  a.k = {static_cast<const uint16_t *>(k), k_row, k_head};
  a.v = {static_cast<const uint16_t *>(v), v_row, v_head};
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.k_lens = k_lens;
  a.out = static_cast<uint16_t *>(out);
  a.lse = lse2;
  a.part = static_cast<float *>(workspace);
  a.err = err;
  a.n_q = n_q;
  a.n_k = n_k;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.n_seqs = n_seqs;
  a.max_q = max_q_per_seq;
  a.max_k = max_k_per_seq;
  a.n_rest = flags & ZX_CROSS_ZERO_REST ? (int32_t)CR_REST : 0;
  a.sm_scale = sm_scale;
  int rc = cr_check("cross_attention", dtype, a, head_dim);
  if (rc) return rc;
  if (n_q == 0) return ZX_OK;
  a.max_q = (int32_t)std::min<int64_t>(max_q_per_seq, n_q);
  cr_group(a);
  ZX_REQUIRE(cu_q && cu_k && out, "cross_attention: null pointer");
  if ((rc = cr_check_rows("cross_attention", "q", a.q, a.group))) return rc;
  if (n_k && ((rc = cr_check_rows("cross_attention", "k", a.k, 1)) || (rc = cr_check_rows("cross_attention", "v", a.v, 1))))
    return rc;
  ZX_REQUIRE(aligned16(out) && aligned16(workspace), "cross_attention: out and workspace must be 16-byte aligned");
  const CrossPlan p = cr_forward_plan(n_seqs, n_kv_heads, a.group, head_dim, a.max_q, max_k_per_seq);
  if (workspace_bytes < cr_forward_bytes(p, n_q, n_q_heads, head_dim) || (!workspace && p.n_split > 1))
    return fail(ZX_ERR_WORKSPACE, "cross_attention: workspace %zu < %zu bytes", workspace_bytes,
                cr_forward_bytes(p, n_q, n_q_heads, head_dim));
  a.n_tile = (int32_t)p.n_tile;
  a.n_split = (int32_t)p.n_split;
  a.order = cr_order(n_seqs, a.max_k / p.n_split, CR_BY_KEYS);
  if (8 * ceil_div((int64_t)n_seqs * n_kv_heads, 8) * p.n_tile * p.n_split >= (1LL << 31) - CR_REST)
    return fail(ZX_ERR_UNSUPPORTED, "cross_attention: too many sequences");
  // q itself is read by the blocks that write there, before they do
  const int64_t width = (int64_t)n_q_heads * head_dim, bytes = 2 * n_q * width;
  const bool in_place = out == q && (n_q == 1 || q_row == width) && (n_q_heads == 1 || q_head == head_dim);
  ZX_REQUIRE(!cr_meets(out, bytes, a.k, n_k, n_kv_heads, head_dim) && !cr_meets(out, bytes, a.v, n_k, n_kv_heads, head_dim),
             "cross_attention: out must not lie in k's or v's memory");
  ZX_REQUIRE(in_place || !cr_meets(out, bytes, a.q, n_q, n_q_heads, head_dim),
             "cross_attention: out must be q itself or not lie in its memory");
  const hipStream_t st = as_stream(stream);
  if (dtype == ZX_BF16) return head_dim == 64 ? cr_forward<CrBf16, 64>(a, p, st) : cr_forward<CrBf16, 128>(a, p, st);
  return head_dim == 64 ? cr_forward<CrF16, 64>(a, p, st) : cr_forward<CrF16, 128>(a, p, st);
}

template <class T, int D>
static int cr_backward(CrossArgs a, const CrossPlan &pq, const CrossPlan &pk, uint16_t *dq, hipStream_t st) {
  int rc;
  a.out = dq;
  a.n_tile = (int32_t)pq.n_tile;
  a.n_split = (int32_t)pq.n_split;
  a.order = cr_order(a.n_seqs, a.max_k / pq.n_split, CR_BY_KEYS);
  cross_dq_kernel<T, D><<<cr_grid(a), CR_THREADS, 0, st>>>(a);
  if ((rc = check_launch("cross_dq"))) return rc;
  const int64_t wq = (int64_t)a.n_q_heads * D, wk = (int64_t)a.n_kv_heads * D;
  if (pq.n_split > 1 && a.n_q) {
    cross_sum_kernel<T><<<(unsigned)ceil_div(a.n_q * wq, 8 * 256), 256, 0, st>>>(a.part, a.n_q * wq, a.n_split, dq, nullptr,
                                                                                a.cu_q, a.n_seqs, a.n_q, wq, a.max_q);
    if ((rc = check_launch("cross_sum"))) return rc;
  }
  if (a.n_k == 0) return ZX_OK;
  a.n_tile = (int32_t)pk.n_tile;
  a.n_split = (int32_t)pk.n_split;
  a.order = cr_order(a.n_seqs, (int64_t)a.max_q * a.group / pk.n_split, CR_BY_ROWS);
  cross_dkv_kernel<T, D><<<cr_grid(a), CR_THREADS, 0, st>>>(a);
  if ((rc = check_launch("cross_dkv")) || pk.n_split == 1) return rc;
  cross_sum_kernel<T><<<dim3((unsigned)ceil_div(a.n_k * wk, 8 * 256), 2), 256, 0, st>>>(
      a.part, 2 * a.n_k * wk, a.n_split, a.dk, a.dv, a.cu_k, a.n_seqs, a.n_k, wk, a.max_k);
  return check_launch("cross_sum");
}

extern "C" int zx_cross_attention_backward(
    int dtype, const void *grad, int64_t g_row, int64_t g_head, const void *q, int64_t n_q, int64_t q_row, int64_t q_head,
    int32_t n_q_heads, const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row, int64_t v_head, int64_t n_k,
    int32_t n_kv_heads, int32_t head_dim, const void *out, const float *lse2, const int32_t *cu_q, const int32_t *cu_k,
    const int32_t *k_lens, int32_t n_seqs, int32_t max_q_per_seq, int32_t max_k_per_seq, float sm_scale, void *dq, void *dk,
    void *dv, int32_t *err, void *workspace, size_t workspace_bytes, zx_stream_t stream) {
  clear_error();
  CrossArgs a = {};
  a.q = {static_cast<const uint16_t *>(q), q_row, q_head};
  a.k = {static_cast<const uint16_t *>(k), k_row, k_head};
  a.v = {static_cast<const uint16_t *>(v), v_row, v_head};
  a.g = {static_cast<const uint16_t *>(grad), g_row, g_head};
  a.o = {static_cast<const uint16_t *>(out), (int64_t)n_q_heads * head_dim, head_dim};
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.k_lens = k_lens;
  a.dk = static_cast<uint16_t *>(dk);
  a.dv = static_cast<uint16_t *>(dv);
  a.lse = const_cast<float *>(lse2);
  a.err = err;
  a.n_q = n_q;
  a.n_k = n_k;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.n_seqs = n_seqs;
  a.max_q = max_q_per_seq;
  a.max_k = max_k_per_seq;
  a.n_rest = (int32_t)CR_REST;
  a.sm_scale = sm_scale;
  int rc = cr_check("cross_attention_backward", dtype, a, head_dim);
  if (rc) return rc;
  a.max_q = (int32_t)std::min<int64_t>(max_q_per_seq, n_q);
  a.max_k = (int32_t)std::min<int64_t>(max_k_per_seq, n_k);
  cr_group(a);
  if (n_q == 0 && n_k == 0) return ZX_OK;
  ZX_REQUIRE(cu_q && cu_k, "cross_attention_backward: null pointer");
  if (n_q && ((rc = cr_check_rows("cross_attention_backward", "q", a.q, a.group)) ||
              (rc = cr_check_rows("cross_attention_backward", "grad", a.g, a.group)) ||
              (rc = cr_check_rows("cross_attention_backward", "out", a.o, a.group))))
    return rc;
  if (n_k && ((rc = cr_check_rows("cross_attention_backward", "k", a.k, 1)) ||
              (rc = cr_check_rows("cross_attention_backward", "v", a.v, 1))))
    return rc;
  ZX_REQUIRE((!n_q || (dq && lse2)) && (!n_k || (dk && dv)), "cross_attention_backward: null pointer");
  ZX_REQUIRE(aligned16(dq) && aligned16(dk) && aligned16(dv) && aligned16(workspace),
             "cross_attention_backward: dq, dk, dv and workspace must be 16-byte aligned");
  const CrossPlan pq = cr_dq_plan(n_seqs, n_kv_heads, a.group, head_dim, a.max_q, a.max_k);
  const CrossPlan pk = cr_dkv_plan(n_seqs, n_kv_heads, a.group, head_dim, a.max_q, a.max_k);
  const CrossGradBytes bytes = cr_grad_bytes(pq, pk, n_q, n_k, n_q_heads, n_kv_heads, head_dim);
  if (workspace_bytes < bytes.delta + bytes.part || (!workspace && bytes.delta + bytes.part))
    return fail(ZX_ERR_WORKSPACE, "cross_attention_backward: workspace %zu < %zu bytes", workspace_bytes,
                bytes.delta + bytes.part);
  a.delta = static_cast<float *>(workspace);
  a.part = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + bytes.delta);
  const int64_t pairs8 = 8 * ceil_div((int64_t)n_seqs * n_kv_heads, 8);
  if (pairs8 * std::max(pq.n_tile * pq.n_split, pk.n_tile * pk.n_split) >= (1LL << 31) - CR_REST)
    return fail(ZX_ERR_UNSUPPORTED, "cross_attention_backward: too many sequences");
  {
    const int64_t wq = (int64_t)n_q_heads * head_dim, wk = (int64_t)n_kv_heads * head_dim;
    struct Rows {
      const CrIn x;
      int64_t n, heads;
    } const of[] = {{a.q, n_q, n_q_heads},  {a.g, n_q, n_q_heads},  {a.o, n_q, n_q_heads},
                    {a.k, n_k, n_kv_heads}, {a.v, n_k, n_kv_heads}, {{a.dk, wk, head_dim}, n_k, n_kv_heads},
                    {{a.dv, wk, head_dim}, n_k, n_kv_heads}};
    bool meets = cr_meets(dk, 2 * n_k * wk, of[6].x, n_k, n_kv_heads, head_dim);
    for (const Rows &r : of) meets = meets || cr_meets(dq, 2 * n_q * wq, r.x, r.n, r.heads, head_dim);
    for (int i = 0; i < 5; ++i)
      for (const void *d : {dk, dv}) meets = meets || cr_meets(d, 2 * n_k * wk, of[i].x, of[i].n, of[i].heads, head_dim);
    ZX_REQUIRE(!meets, "cross_attention_backward: dq, dk and dv must not lie in each other's memory or the inputs'");
  }
  const hipStream_t st = as_stream(stream);
  uint16_t *d = static_cast<uint16_t *>(dq);
  if (dtype == ZX_BF16)
    return head_dim == 64 ? cr_backward<CrBf16, 64>(a, pq, pk, d, st) : cr_backward<CrBf16, 128>(a, pq, pk, d, st);
  return head_dim == 64 ? cr_backward<CrF16, 64>(a, pq, pk, d, st) : cr_backward<CrF16, 128>(a, pq, pk, d, st);
}
