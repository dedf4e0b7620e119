// Attention over long rows (no counterpart in the reference, whose longest row is a few dozen tokens: mgcvae.py:276-282,375-449):
//   mmt_long_attention_fwd / _bwd   capped scores, distance bias, learned bucket bias, document / prefix / causal masks, cache
//                                   lengths, shared key heads; bf16, fp16, fp32; forward, backward, few rows over a long cache
// mmt_attention_fwd / _bwd (train.hip) stay the path for rows of at most 32 keys with stored probabilities.
#include "long_attention.cuh"

#include <algorithm>

int mmt_set_error(int code, const char *fmt, ...);   // transformer.hip

namespace la {

struct Args {                      // mmt_long_attention plus what the launcher derives
  mmt_long_attention a;
  int G, pack;                     // query heads per key head; heads sharing a workgroup's rows (1 or G)
  int nqt, nkt, nsplit, items;     // row tiles, key tiles, splits of the keys, work items
  const DocRange *krng, *qrng;     // per batch row and tile, or NULL
  void *out;                       // (B, Lq, H, dh)
  float *lse;                      // (B, H, Lq)
  float *part_o;                   // split: (nsplit, B, H, Lq, dh)
  float *part_ml;                  // split: (nsplit, B, H, Lq, 2): maximum, sum
  // backward
  const void *dout;
  int64_t do_bs, do_rs, do_hs;
  const float2 *stat;              // (B, H, Lq): lse in units of log 2, rowsum(do o) - dlse
  const float *dscale;             // fp16: power of two the score gradients are multiplied by before they are rounded
  void *dq, *dk, *dv;              // (B, Lq, H, dh), (B, Lk, Hk, dh)
  const float *dlse;               // (B, H, Lq) gradient of the log-sum, or NULL
  float *delta_fix;                // (B, H, Lq) delta with the exact rowsum(P dP), or NULL
  float *far_part;                 // (items, 2)
};

// what a lane knows about its query row
struct Row {
  bool valid, live;                // a row of this call; and not padding
  int i, h, p, hi, doc;            // query, head, position, first invisible key (before documents), document
  float slope;                     // slope times log2 e
};

template <typename A> __device__ __forceinline__ int row_len(const A &a, int b) {
  return a.kv_len ? max(0, min(a.kv_len[b], a.Lk)) : a.Lk;
}

__device__ __forceinline__ Row make_row(const Args &g, int b, int head0, int r, int len) {
  const mmt_long_attention &a = g.a;
  Row w;
  w.i = r / g.pack;
  w.h = head0 + r % g.pack;
  w.valid = w.i < a.Lq;
  w.p = len - a.Lq + w.i;
  w.doc = 0;
  if (a.q_doc && w.valid) w.doc = a.q_doc[(int64_t)b * a.Lq + w.i];
  w.live = w.valid && w.doc >= 0;
  w.hi = len;
  if (a.causal) w.hi = min(len, max(w.p + 1, a.prefix ? a.prefix[b] : 0));
  w.slope = a.slopes && w.valid ? a.slopes[w.h] * LOG2E : 0.f;
  return w;
}

// bounds over the live rows of a wave, then of the workgroup
struct Bounds {
  int hi_min, hi_max, p_min, p_max, d_min, d_max;
};
__device__ __forceinline__ Bounds wave_bounds(const Row &w) {
  Bounds b;
  b.hi_min = wave_min(w.live ? w.hi : 0x7fffffff);
  b.hi_max = wave_max(w.live ? w.hi : 0);
  b.p_min = wave_min(w.live ? w.p : 0x7fffffff);
  b.p_max = wave_max(w.live ? w.p : -0x7fffffff);
  b.d_min = wave_min(w.live ? w.doc : 0x7fffffff);
  b.d_max = wave_max(w.live ? w.doc : -1);
  return b;
}
__device__ __forceinline__ Bounds group_bounds(const Bounds &w, int *s, int wave) {      // s: 6 * WAVES ints of LDS
  if ((threadIdx.x & 63) == 0) {
    s[wave * 6 + 0] = w.hi_min, s[wave * 6 + 1] = w.hi_max, s[wave * 6 + 2] = w.p_min;
    s[wave * 6 + 3] = w.p_max, s[wave * 6 + 4] = w.d_min, s[wave * 6 + 5] = w.d_max;
  }
  __syncthreads();
  Bounds b = {0x7fffffff, 0, 0x7fffffff, -0x7fffffff, 0x7fffffff, -1};
  for (int v = 0; v < WAVES; ++v) {
    b.hi_min = min(b.hi_min, s[v * 6 + 0]), b.hi_max = max(b.hi_max, s[v * 6 + 1]), b.p_min = min(b.p_min, s[v * 6 + 2]);
    b.p_max = max(b.p_max, s[v * 6 + 3]), b.d_min = min(b.d_min, s[v * 6 + 4]), b.d_max = max(b.d_max, s[v * 6 + 5]);
  }
  b.hi_min = __builtin_amdgcn_readfirstlane(b.hi_min), b.hi_max = __builtin_amdgcn_readfirstlane(b.hi_max);
  b.p_min = __builtin_amdgcn_readfirstlane(b.p_min), b.p_max = __builtin_amdgcn_readfirstlane(b.p_max);
  b.d_min = __builtin_amdgcn_readfirstlane(b.d_min), b.d_max = __builtin_amdgcn_readfirstlane(b.d_max);
  return b;
}

// The learned bias in LDS: the table rows of the workgroup's heads (in units of log 2) and the bucket of each clamped distance.
// Bucket numbers outside the table are clamped into it.  An entry at or below -2^100 (the lowest value of a type, used as a mask) is
// taken for -inf: next to it a score vanishes in rounding, and the saved log-sum of a row of such entries could not tell them apart.
struct BiasLds {
  float *table;             // [pack][nb]
  unsigned char *bucket;    // [2 reach + 1]
  __device__ __forceinline__ void fill(const mmt_long_attention &a, int head0, int pack) {
    for (int n = threadIdx.x; n < pack * a.n_buckets; n += THREADS) {
      const float v = a.rel_bias[(int64_t)(head0 + n / a.n_buckets) * a.n_buckets + n % a.n_buckets];
      table[n] = v <= -0x1p100f ? -INFINITY : v * LOG2E;
    }
    for (int n = threadIdx.x; n < 2 * a.reach + 1; n += THREADS)
      bucket[n] = (unsigned char)max(0, min(a.rel_buckets[n], a.n_buckets - 1));
  }
};
static inline __host__ __device__ int bias_lds_bytes(const mmt_long_attention &a, int pack) {
  return a.rel_bias ? pack * a.n_buckets * 4 + ((2 * a.reach + 1 + 15) & ~15) : 0;
}

// A lane's N scores of one key tile (raw products s) -> u in units of log 2; what the row cannot see becomes -inf.
// `t` receives tanh(s / cap) when the scores are capped and the caller needs it.
// Returns the factor that still has to be applied to x (scale log2 e on the plain path, which leaves the products alone).
struct ScoreCtx {
  float c_scale, cap_in, cap_out;  // scale log2 e; scale / cap; cap log2 e
  bool capped, biased, rel;
};
__device__ __forceinline__ ScoreCtx score_ctx(const mmt_long_attention &a) {
  ScoreCtx s;
  s.c_scale = a.scale * LOG2E;
  s.capped = a.softcap > 0.f;
  s.cap_in = s.capped ? a.scale / a.softcap : 0.f;
  s.cap_out = a.softcap * LOG2E;
  s.rel = a.rel_bias != nullptr;
  s.biased = s.rel || a.slopes != nullptr;
  return s;
}

template <int N, bool KEEP>
__device__ __forceinline__ float transform(const mmt_long_attention &a, const ScoreCtx &sc, float *x, float *t, int key0, int h, int p, float slope,
                                           const float *tab, const unsigned char *bucket, int far, bool need_mask, int hi, int doc,
                                           const int *kdoc) {
  float c = sc.c_scale;
  if (sc.capped) {
    tanh_scores<N>(x, sc.cap_in);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (KEEP) t[i] = x[i];
      x[i] *= sc.cap_out;
    }
    c = 1.f;
  } else if (sc.biased) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= c;
    c = 1.f;
  }
  if (sc.biased) {
    const int d0 = key0 + 4 * h - p;
    if (a.slopes) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = fmaf(-slope, fabsf((float)(d0 + 8 * (i >> 2) + (i & 3))), x[i]);
    }
    if (sc.rel) {
      if (far != 0) {                                   // the whole tile lies beyond the reach: one bucket
        const float v = tab[bucket[far < 0 ? 0 : 2 * a.reach]];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] += v;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int d = max(-a.reach, min(a.reach, d0 + 8 * (i >> 2) + (i & 3))) + a.reach;
          x[i] += tab[bucket[d]];
        }
      }
    }
  }
  if (need_mask) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = 8 * (i >> 2) + 4 * h + (i & 3);
      bool see = key0 + j < hi;
      if (kdoc) see = see && kdoc[j] == doc;
      if (!see) x[i] = -INFINITY;
    }
  }
  return c;
}

// ---------------------------------------------------------------------------------------------------------------- forward
// One workgroup = 128 rows (4 waves x 32) of one head - or of the `pack` heads that share a key head, when there are few queries -
// against a range of key tiles.  K and V tiles go memory -> registers -> LDS one tile ahead of the products.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_fwd_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BK = L::BK, NK = BK / 32, NC = D / 16, ND = D / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  char *sK = smem, *sV = smem + L::BYTES;
  int *sDoc = (int *)(smem + 2 * L::BYTES), *sB = sDoc + BK;
  BiasLds bias;
  bias.table = (float *)(sB + 6 * WAVES);
  const int item = xcd_item(g.items);
  if (item < 0) return;
  const int split = item % g.nsplit;
  int n = item / g.nsplit;
  const int ngroup = g.pack > 1 ? 1 : g.G;
  const int gi = n % ngroup;
  n /= ngroup;
  int qt = n % g.nqt;
  if (a.causal) qt = g.nqt - 1 - qt;                     // the tiles with the most keys first
  n /= g.nqt;
  const int kh = n % a.Hk, b = n / a.Hk;
  const int head0 = kh * g.G + gi;
  bias.bucket = (unsigned char *)(bias.table + (a.rel_bias ? g.pack * a.n_buckets : 0));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b);
  const Row w = make_row(g, b, head0, qt * ROWS + wave * 32 + col, len);
  const Bounds wb = wave_bounds(w);
  const Bounds gb = group_bounds(wb, sB, wave);
  if (a.rel_bias) bias.fill(a, head0, g.pack);
  const float *tab = bias.table + (g.pack > 1 ? (w.h - head0) * a.n_buckets : 0);

  const T *qrow = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)min(w.i, a.Lq - 1) * a.q_rs + (int64_t)w.h * a.q_hs;
  V8 fq[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) fq[c] = mem_frag<T>(qrow, c, h, a.dh, w.live);

  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  float m = -INFINITY, l = 0.f;
  const ScoreCtx sc = score_ctx(a);

  const int tiles = (gb.hi_max + BK - 1) / BK, per = (tiles + g.nsplit - 1) / g.nsplit;
  const DocRange *rng = g.krng ? g.krng + (int64_t)b * g.nkt : nullptr;
  TileIter it;
  it.start(rng, gb.d_min, gb.d_max, split * per, min(tiles, (split + 1) * per));
  const T *kbase = (const T *)a.k + (int64_t)b * a.k_bs + (int64_t)kh * a.k_hs;
  const T *vbase = (const T *)a.v + (int64_t)b * a.v_bs + (int64_t)kh * a.v_hs;
  const int *kdoc = a.k_doc ? a.k_doc + (int64_t)b * a.Lk : nullptr;
  Stage<T, D> stk, stv;
  int t = it.next();
  if (t >= 0) {
    stk.load(kbase, a.k_rs, t * BK, a.Lk, a.dh);
    stv.load(vbase, a.v_rs, t * BK, a.Lk, a.dh);
  }
  while (t >= 0) {
    const int k0 = t * BK;
    __syncthreads();
    stk.store(sK, k0, len, kdoc);
    stv.store(sV, k0, len, kdoc);
    if (kdoc && threadIdx.x < BK) sDoc[threadIdx.x] = k0 + (int)threadIdx.x < a.Lk ? kdoc[k0 + threadIdx.x] : -1;
    const bool one_doc = !rng || (rng[t].dead == 0 && rng[t].lo == rng[t].hi && wb.d_min == wb.d_max && wb.d_min == rng[t].lo);
    const int tn = it.next();
    if (tn >= 0) {
      stk.load(kbase, a.k_rs, tn * BK, a.Lk, a.dh);
      stv.load(vbase, a.v_rs, tn * BK, a.Lk, a.dh);
    }
    __syncthreads();
    if (k0 < wb.hi_max) {
      const bool need_mask = k0 + BK > wb.hi_min || !one_doc;
      const int far = !a.rel_bias ? 0 : k0 + BK - 1 - wb.p_min <= -a.reach ? -1 : k0 - wb.p_max >= a.reach ? 1 : 0;
      float x[NK * 16];
#pragma unroll
      for (int kt = 0; kt < NK; ++kt) {
        f32x16 s = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) s = Elem<T>::mma(row_frag<T, D>(sK, 32 * kt + col, c, h), fq[c], s);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[16 * kt + i] = s[i];
      }
      float cf = 1.f;
#pragma unroll
      for (int kt = 0; kt < NK; ++kt)
        cf = transform<16, false>(a, sc, x + 16 * kt, nullptr, k0 + 32 * kt, h, w.p, w.slope, tab, bias.bucket, far, need_mask, w.hi, w.doc,
                                  kdoc ? sDoc + 32 * kt : nullptr);
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < NK * 16; ++i) mx = fmaxf(mx, x[i]);
      const float m_new = fmaxf(m, half_max(mx) * cf);
      const float ms = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = ex2(m - ms);
      m = m_new;
      const float off = Elem<T>::PSHIFT - ms;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NK * 16; ++i) {
        x[i] = ex2(fmaf(x[i], cf, off));
        sum += x[i];
      }
      l = fmaf(l, alpha, sum);
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
      }
#pragma unroll
      for (int c = 0; c < NK * 2; ++c) {
        const V8 p = round8<T>(x + 8 * c);
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = Elem<T>::mma(col_frag<T, D>(sV, 16 * c, d, lane), p, acc[d]);
      }
    }
    t = tn;
  }
  l = half_sum(l);
  if (!w.valid) return;
  const int64_t r = ((int64_t)b * a.H + w.h) * a.Lq + w.i;
  if (g.nsplit > 1) {
    const int64_t rs = (int64_t)split * a.B * a.H * a.Lq + r;
    if (h == 0) {
      g.part_ml[2 * rs] = w.live ? m : -INFINITY;
      g.part_ml[2 * rs + 1] = w.live ? l : 0.f;
    }
    float *o = g.part_o + rs * a.dh;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int dim = 32 * d + 8 * q + 4 * h;
        if (dim < a.dh) *(f32x4 *)(o + dim) = f32x4{acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]};
      }
    return;
  }
  const bool some = w.live && l != 0.f;                   // (a NaN sum is "some")
  const float inv = some ? 1.f / l : 0.f;
  if (g.lse && h == 0) g.lse[r] = some ? (m + log2f(l) - Elem<T>::PSHIFT) * LN2 : -INFINITY;
  T *o = (T *)g.out + (((int64_t)b * a.Lq + w.i) * a.H + w.h) * a.dh;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dim = 32 * d + 8 * q + 4 * h;
      if (dim < a.dh) {
        typename Elem<T>::V4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(some ? acc[d][4 * q + e] * inv : 0.f);
        *(typename Elem<T>::V4 *)(o + dim) = v;
      }
    }
}

// Joins the splits of a row: weights 2^(m_s - max m).  16 lanes per row, up to 8 elements per lane.
template <typename T> __global__ void __launch_bounds__(256) mmt_long_attn_join_kernel(const Args g) {
  const mmt_long_attention &a = g.a;
  const int64_t rows = (int64_t)a.B * a.H * a.Lq, r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (r >= rows) return;
  const int d0 = (threadIdx.x & 15) * 8;
  float m = -INFINITY;
  for (int s = 0; s < g.nsplit; ++s) m = fmaxf(m, g.part_ml[2 * (s * rows + r)]);
  const float ms = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 o[2] = {};
  for (int s = 0; s < g.nsplit; ++s) {
    const int64_t rs = s * rows + r;
    const float ls = g.part_ml[2 * rs + 1], f = ls == 0.f ? 0.f : ex2(g.part_ml[2 * rs] - ms);
    l = fmaf(ls, f, l);
    if (d0 < a.dh && ls != 0.f) {
      o[0] += *(const f32x4 *)(g.part_o + rs * a.dh + d0) * f;
      o[1] += *(const f32x4 *)(g.part_o + rs * a.dh + d0 + 4) * f;
    }
  }
  const bool some = l != 0.f;
  const float inv = some ? 1.f / l : 0.f;
  const int64_t i = r % a.Lq, bh = r / a.Lq, hd = bh % a.H, b = bh / a.H;
  if (g.lse && (threadIdx.x & 15) == 0) g.lse[r] = some ? (m + log2f(l) - Elem<T>::PSHIFT) * LN2 : -INFINITY;
  if (d0 < a.dh) {
    typename Elem<T>::V8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)(some ? o[e >> 2][e & 3] * inv : 0.f);
    *(typename Elem<T>::V8 *)((T *)g.out + ((b * a.Lq + i) * a.H + hd) * a.dh + d0) = v;
  }
}

// document ids -> per tile of `bk`: smallest, largest live id, and whether any row of the tile is dead or missing
__global__ void mmt_long_attn_docs_kernel(const int *doc, int L, int nt, int bk, int total, DocRange *out) {
  const int n = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= total) return;
  const int64_t b = n / nt;
  const int t = n % nt, j = t * bk + lane;
  const int id = lane < bk && j < L ? doc[b * L + j] : -1;
  const int lo = wave_min(id >= 0 ? id : 0x7fffffff), hi = wave_max(id);
  const bool dead = __any(lane < bk && id < 0);
  if (lane == 0) out[n] = DocRange{lo, hi, dead ? 1 : 0, 0};
}

// --------------------------------------------------------------------------------------------------------------- backward
//   dV = P^T dO;   dP = dO V^T;   dU = P (dP - delta), delta_i = rowsum(dO o) - dlse_i;   dS = dU (1 - tanh^2)
//   dQ = scale dS K;   dK = scale dS^T Q;   dtable[h][b] = sum of dU over the pairs of the bucket
// Two kernels recompute the probabilities from the saved log-sum: one walks the keys of a query tile (dQ), the other the queries of
// a key tile (dK, dV, summed over the query heads that share the key head).  Seven products instead of the five of a single pass,
// but every sum has a fixed order and an owner: no atomics, the same bits every time.

// fp16: the score gradients are rounded to 5 exponent bits, so they are first multiplied by a power of two that takes their bound
// 2 max|do_i| max|v_j| + max|dlse| to at most 2^15.  maxima: bits of max|do|^2, max|v|^2, max|dlse| (non-negative floats order like
// integers; an integer maximum does not depend on the order of the workgroups)
__global__ void mmt_long_attn_zero_kernel(unsigned *w, int n) {
  if ((int)threadIdx.x < n) w[threadIdx.x] = 0;
}
template <typename T> __global__ void __launch_bounds__(256) mmt_long_attn_vnorm_kernel(const Args g, unsigned *maxima) {
  const mmt_long_attention &a = g.a;
  const int64_t rows = (int64_t)a.B * a.Lk * a.Hk;
  float mx = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); r < rows; r += (int64_t)gridDim.x * 16) {
    const int64_t hd = r % a.Hk, bj = r / a.Hk, j = bj % a.Lk, b = bj / a.Lk;
    if (j >= row_len(a, (int)b) || (a.k_doc && a.k_doc[b * a.Lk + j] < 0)) continue;
    const int d0 = (threadIdx.x & 15) * 8;
    float s = 0.f;
    if (d0 < a.dh) {
      const typename Elem<T>::V8 v = *(const typename Elem<T>::V8 *)((const T *)a.v + b * a.v_bs + j * a.v_rs + hd * a.v_hs + d0);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf((float)v[e], (float)v[e], s);
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) s += __shfl_xor(s, m);
    if (isfinite(s)) mx = fmaxf(mx, s);
  }
#pragma unroll
  for (int m = 16; m < 64; m <<= 1) mx = fmaxf(mx, __shfl_xor(mx, m));
  if ((threadIdx.x & 63) == 0) atomicMax(maxima + 1, __float_as_uint(mx));
}
__global__ void mmt_long_attn_dscale_kernel(const unsigned *maxima, float *dscale) {
  const float nd = sqrtf(__uint_as_float(maxima[0])), nv = sqrtf(__uint_as_float(maxima[1])), nl = __uint_as_float(maxima[2]);
  const float bound = 2.f * nd * nv + nl;
  int e = 0;
  const bool known = bound > 0.f && isfinite(bound);
  if (known) (void)frexpf(bound, &e);                                     // bound < 2^e
  dscale[0] = ldexpf(1.f, known ? max(-60, min(60, 15 - e)) : 0);
}

// delta and the log-sum in units of log 2; 16 lanes per row
template <typename T> __global__ void __launch_bounds__(256) mmt_long_attn_stat_kernel(const Args g, const float *dlse, float2 *stat, unsigned *maxima) {
  const mmt_long_attention &a = g.a;
  const int64_t rows = (int64_t)a.B * a.H * a.Lq;
  float mx = 0.f, ml = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); r < rows; r += (int64_t)gridDim.x * 16) {
    // rows in the order of the tensors (b, i, h), the statistics in the order of the kernels that read them (b, h, i)
    const int64_t hd = r % a.H, bi = r / a.H, i = bi % a.Lq, b = bi / a.Lq, w = (b * a.H + hd) * a.Lq + i;
    const int d0 = (threadIdx.x & 15) * 8;
    const bool live = !(a.q_doc && a.q_doc[b * a.Lq + i] < 0);
    float s = 0.f, nn = 0.f;
    if (d0 < a.dh && live) {
      const typename Elem<T>::V8 o = *(const typename Elem<T>::V8 *)((const T *)g.out + r * a.dh + d0);
      const typename Elem<T>::V8 d = *(const typename Elem<T>::V8 *)((const T *)g.dout + b * g.do_bs + i * g.do_rs + hd * g.do_hs + d0);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s = fmaf((float)o[e], (float)d[e], s);
        nn = fmaf((float)d[e], (float)d[e], nn);
      }
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
      s += __shfl_xor(s, m);
      nn += __shfl_xor(nn, m);
    }
    const float ls = g.lse[w], dl = dlse && live ? dlse[w] : 0.f;
    if (isfinite(nn)) mx = fmaxf(mx, nn);
    if (isfinite(dl)) ml = fmaxf(ml, fabsf(dl));
    // a row without keys has probabilities 0: its log-sum is turned around
    if ((threadIdx.x & 15) == 0) stat[w] = make_float2(ls == -INFINITY ? INFINITY : ls * LOG2E, s - dl);
  }
  if (!maxima) return;
#pragma unroll
  for (int m = 16; m < 64; m <<= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, m));
    ml = fmaxf(ml, __shfl_xor(ml, m));
  }
  if ((threadIdx.x & 63) == 0) {
    atomicMax(maxima, __float_as_uint(mx));
    atomicMax(maxima + 2, __float_as_uint(ml));
  }
}

// dQ.  The forward's geometry; K is read twice from LDS (as rows for the scores, transposed for dQ^T += K^T dS^T), V once.
// With a learned bias it also leaves, per row, the exact delta (see the table kernel) and the sums of dU over the tiles that lie wholly
// beyond the reach on either side.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_dq_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BK = L::BK, NK = BK / 32, NC = D / 16, ND = D / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  char *sK = smem, *sV = smem + L::BYTES;
  int *sDoc = (int *)(smem + 2 * L::BYTES), *sB = sDoc + BK;
  BiasLds bias;
  bias.table = (float *)(sB + 6 * WAVES);
  bias.bucket = (unsigned char *)(bias.table + (a.rel_bias ? a.n_buckets : 0));
  const int item = xcd_item(g.items);
  if (item < 0) return;
  int n = item;
  const int gi = n % g.G;
  n /= g.G;
  int qt = n % g.nqt;
  if (a.causal) qt = g.nqt - 1 - qt;
  n /= g.nqt;
  const int kh = n % a.Hk, b = n / a.Hk, head = kh * g.G + gi;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b);
  const Row w = make_row(g, b, head, qt * ROWS + wave * 32 + col, len);
  const Bounds wb = wave_bounds(w);
  const Bounds gb = group_bounds(wb, sB, wave);
  if (a.rel_bias) bias.fill(a, head, 1);
  const int64_t r = ((int64_t)b * a.H + head) * a.Lq + min(w.i, a.Lq - 1);
  const float2 st = w.live ? g.stat[r] : make_float2(INFINITY, 0.f);

  const T *qrow = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)min(w.i, a.Lq - 1) * a.q_rs + (int64_t)head * a.q_hs;
  const T *drow = (const T *)g.dout + (int64_t)b * g.do_bs + (int64_t)min(w.i, a.Lq - 1) * g.do_rs + (int64_t)head * g.do_hs;
  V8 fq[NC], fd[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    fq[c] = mem_frag<T>(qrow, c, h, a.dh, w.live);
    fd[c] = mem_frag<T>(drow, c, h, a.dh, w.live);
  }
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  const ScoreCtx sc = score_ctx(a);
  const float dscale = sizeof(T) == 2 && g.dscale ? g.dscale[0] : 1.f;
  float all_u = 0.f, far_u[2] = {0.f, 0.f}, far_p[2] = {0.f, 0.f};

  const int tiles = (gb.hi_max + BK - 1) / BK;
  const DocRange *rng = g.krng ? g.krng + (int64_t)b * g.nkt : nullptr;
  TileIter it;
  it.start(rng, gb.d_min, gb.d_max, 0, tiles);
  const T *kbase = (const T *)a.k + (int64_t)b * a.k_bs + (int64_t)kh * a.k_hs;
  const T *vbase = (const T *)a.v + (int64_t)b * a.v_bs + (int64_t)kh * a.v_hs;
  const int *kdoc = a.k_doc ? a.k_doc + (int64_t)b * a.Lk : nullptr;
  Stage<T, D> stk, stv;
  int t = it.next();
  if (t >= 0) {
    stk.load(kbase, a.k_rs, t * BK, a.Lk, a.dh);
    stv.load(vbase, a.v_rs, t * BK, a.Lk, a.dh);
  }
  while (t >= 0) {
    const int k0 = t * BK;
    __syncthreads();
    stk.store(sK, k0, len, kdoc);
    stv.store(sV, k0, len, kdoc);
    if (kdoc && threadIdx.x < BK) sDoc[threadIdx.x] = k0 + (int)threadIdx.x < a.Lk ? kdoc[k0 + threadIdx.x] : -1;
    const bool one_doc = !rng || (rng[t].dead == 0 && rng[t].lo == rng[t].hi && wb.d_min == wb.d_max && wb.d_min == rng[t].lo);
    const int tn = it.next();
    if (tn >= 0) {
      stk.load(kbase, a.k_rs, tn * BK, a.Lk, a.dh);
      stv.load(vbase, a.v_rs, tn * BK, a.Lk, a.dh);
    }
    __syncthreads();
    if (k0 < wb.hi_max) {
      const bool need_mask = k0 + BK > wb.hi_min || !one_doc;
      // by the whole workgroup's rows: the table kernel takes the tiles that are left with the same rule
      const int far = !a.rel_bias ? 0 : k0 + BK - 1 - gb.p_min <= -a.reach ? -1 : k0 - gb.p_max >= a.reach ? 1 : 0;
#pragma unroll
      for (int kt = 0; kt < NK; ++kt) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s = Elem<T>::mma(row_frag<T, D>(sK, 32 * kt + col, c, h), fq[c], s);
          dp = Elem<T>::mma(row_frag<T, D>(sV, 32 * kt + col, c, h), fd[c], dp);
        }
        float x[16], th[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = s[i];
        const float cf = transform<16, true>(a, sc, x, th, k0 + 32 * kt, h, w.p, w.slope, bias.table, bias.bucket, far, need_mask, w.hi,
                                             w.doc, kdoc ? sDoc + 32 * kt : nullptr);
        float su = 0.f, sp = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = ex2(fmaf(x[i], cf, -st.x));
          x[i] = p * (dp[i] - st.y);
          if (p == 0.f) x[i] = 0.f;                       // a key that the row does not see may hold anything
          su += x[i];
          sp += p;
        }
        if (a.rel_bias) {
          all_u += su;
          if (far != 0) {
            far_u[far > 0] += su;
            far_p[far > 0] += sp;
          }
        }
        if (sc.capped) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= fmaf(-th[i], th[i], 1.f);
        }
        if (sizeof(T) == 2 && Elem<T>::PSHIFT != 0.f) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= dscale;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const V8 ds = round8<T>(x + 8 * c);
#pragma unroll
          for (int d = 0; d < ND; ++d) acc[d] = Elem<T>::mma(col_frag<T, D>(sK, 32 * kt + 16 * c, d, lane), ds, acc[d]);
        }
      }
    }
    t = tn;
  }
  if (a.rel_bias) {
    // the sum of dU over a row is dlse (0 without it) by definition: what is left is what the rounding of o has put into delta
    all_u = half_sum(all_u) - (g.dlse && w.live ? g.dlse[r] : 0.f);
    if (w.valid && h == 0) g.delta_fix[r] = st.y + (w.live ? all_u : 0.f);
    if (!w.live) all_u = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) far_u[s] = wave_sum(w.live ? far_u[s] - all_u * far_p[s] : 0.f);
    __syncthreads();
    float *sF = (float *)sB;
    if (lane == 0) sF[2 * wave] = far_u[0], sF[2 * wave + 1] = far_u[1];
    __syncthreads();
    if (threadIdx.x < 2) {
      float v = 0.f;
      for (int u = 0; u < WAVES; ++u) v += sF[2 * u + threadIdx.x];
      // item order (b, qt, head) for the reduction, whatever order the workgroups ran in
      g.far_part[(((int64_t)b * g.nqt + qt) * a.H + head) * 2 + threadIdx.x] = v;
    }
  }
  if (!w.valid) return;
  T *o = (T *)g.dq + (((int64_t)b * a.Lq + w.i) * a.H + head) * a.dh;
  const float f = a.scale / dscale;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dim = 32 * d + 8 * q + 4 * h;
      if (dim < a.dh) {
        typename Elem<T>::V4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(w.live ? acc[d][4 * q + e] * f : 0.f);
        *(typename Elem<T>::V4 *)(o + dim) = v;
      }
    }
}

// dK, dV.  A wave owns 32 keys (the accumulator's columns; their rows of K and V stay in registers as operands), the queries of all
// heads that share the key head go by in LDS tiles, as rows for S and dP and transposed for dV^T += dO^T P and dK^T += Q^T dS.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_dkv_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BQ = L::BK, NQ = BQ / 32, NC = D / 16, ND = D / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  char *sQ = smem, *sO = smem + L::BYTES;
  float2 *sStat = (float2 *)(smem + 2 * L::BYTES);
  int *sDoc = (int *)(sStat + BQ), *sB = sDoc + BQ;
  BiasLds bias;
  bias.table = (float *)(sB + 6 * WAVES);
  bias.bucket = (unsigned char *)(bias.table + (a.rel_bias ? g.G * a.n_buckets : 0));
  const int item = xcd_item(g.items);
  if (item < 0) return;
  int n = item;
  const int kt = n % ((a.Lk + ROWS - 1) / ROWS);          // causal: the first keys are seen by the most queries
  n /= (a.Lk + ROWS - 1) / ROWS;
  const int kh = n % a.Hk, b = n / a.Hk, head0 = kh * g.G;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b), off = len - a.Lq, prefix = a.prefix ? a.prefix[b] : 0;
  const int j = kt * ROWS + wave * 32 + col;
  const int kdoc = a.k_doc && j < a.Lk ? a.k_doc[(int64_t)b * a.Lk + j] : 0;
  const bool live = j < len && kdoc >= 0;
  const int j_lo = kt * ROWS + wave * 32;                 // first key of the wave
  const int d_min = wave_min(live ? kdoc : 0x7fffffff), d_max = wave_max(live ? kdoc : -1);
  const bool all_live = __all(live);
  if (lane == 0) sB[2 * wave] = d_min, sB[2 * wave + 1] = d_max;
  __syncthreads();
  int gd_min = 0x7fffffff, gd_max = -1;
  for (int v = 0; v < WAVES; ++v) gd_min = min(gd_min, sB[2 * v]), gd_max = max(gd_max, sB[2 * v + 1]);
  if (a.rel_bias) bias.fill(a, head0, g.G);

  const T *krow = (const T *)a.k + (int64_t)b * a.k_bs + (int64_t)min(j, a.Lk - 1) * a.k_rs + (int64_t)kh * a.k_hs;
  const T *vrow = (const T *)a.v + (int64_t)b * a.v_bs + (int64_t)min(j, a.Lk - 1) * a.v_rs + (int64_t)kh * a.v_hs;
  V8 fk[NC], fv[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    fk[c] = mem_frag<T>(krow, c, h, a.dh, live);
    fv[c] = mem_frag<T>(vrow, c, h, a.dh, live);
  }
  f32x16 acck[ND], accv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acck[d] = f32x16{}, accv[d] = f32x16{};
  const ScoreCtx sc = score_ctx(a);
  // fp16: P is rounded times 2^PSHIFT; the surplus is taken out of dS again together with its own scaling
  const float dscale = sizeof(T) == 2 && g.dscale ? g.dscale[0] : 1.f;
  const float ds_mul = dscale * ex2(-Elem<T>::PSHIFT);

  // queries that may see a key of this workgroup: position >= its first key, unless the prefix reaches into it
  const int i_first = a.causal && prefix <= kt * ROWS ? max(0, kt * ROWS - off) : 0;
  const int t0 = i_first / BQ, t1 = kt * ROWS < len ? (a.Lq + BQ - 1) / BQ : 0;
  const DocRange *rng = g.qrng ? g.qrng + (int64_t)b * ((a.Lq + BQ - 1) / BQ) : nullptr;
  const int *qdoc = a.q_doc ? a.q_doc + (int64_t)b * a.Lq : nullptr;
  for (int gi = 0; gi < g.G; ++gi) {
    const int head = head0 + gi;
    const float slope = a.slopes ? a.slopes[head] * LOG2E : 0.f;
    const float *tab = bias.table + gi * a.n_buckets;
    const T *qbase = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)head * a.q_hs;
    const T *dbase = (const T *)g.dout + (int64_t)b * g.do_bs + (int64_t)head * g.do_hs;
    const float2 *stat = g.stat + ((int64_t)b * a.H + head) * a.Lq;
    TileIter it;
    it.start(rng, gd_min, gd_max, t0, t1);
    Stage<T, D> stq, std;
    int t = it.next();
    if (t >= 0) {
      stq.load(qbase, a.q_rs, t * BQ, a.Lq, a.dh);
      std.load(dbase, g.do_rs, t * BQ, a.Lq, a.dh);
    }
    while (t >= 0) {
      const int q0 = t * BQ;
      __syncthreads();
      stq.store(sQ, q0, a.Lq, qdoc);
      std.store(sO, q0, a.Lq, qdoc);
      if (threadIdx.x < BQ) {
        const int i = q0 + threadIdx.x;
        const int id = i < a.Lq ? (qdoc ? qdoc[i] : 0) : -1;
        sDoc[threadIdx.x] = id;
        sStat[threadIdx.x] = id >= 0 ? stat[i] : make_float2(INFINITY, 0.f);
      }
      const bool one_doc = !rng || (rng[t].dead == 0 && rng[t].lo == rng[t].hi && d_min == d_max && d_min == rng[t].lo);
      const int tn = it.next();
      if (tn >= 0) {
        stq.load(qbase, a.q_rs, tn * BQ, a.Lq, a.dh);
        std.load(dbase, g.do_rs, tn * BQ, a.Lq, a.dh);
      }
      __syncthreads();
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt) {
        const int i0 = q0 + 32 * qt, p0 = off + i0;
        // the last row of the sub-tile sees the most
        if (a.causal && max(p0 + 32, prefix) <= j_lo) continue;
        const bool need_mask = !one_doc || !all_live || (a.causal && max(p0 + 1, prefix) < j_lo + 32);
        const int far = !a.rel_bias ? 0 : j_lo + 31 - p0 <= -a.reach ? -1 : j_lo - (p0 + 31) >= a.reach ? 1 : 0;
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s = Elem<T>::mma(row_frag<T, D>(sQ, 32 * qt + col, c, h), fk[c], s);
          dp = Elem<T>::mma(row_frag<T, D>(sO, 32 * qt + col, c, h), fv[c], dp);
        }
        float x[16], th[16];
        float cf = sc.c_scale;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = s[i];
        if (sc.capped) {
          tanh_scores<16>(x, sc.cap_in);
#pragma unroll
          for (int i = 0; i < 16; ++i) th[i] = x[i], x[i] *= sc.cap_out;
          cf = 1.f;
        } else if (sc.biased) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= cf;
          cf = 1.f;
        }
        if (sc.biased) {
          const int d0 = j - p0 - 4 * h;
          if (a.slopes) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fmaf(-slope, fabsf((float)(d0 - 8 * (i >> 2) - (i & 3))), x[i]);
          }
          if (sc.rel) {
            if (far != 0) {
              const float v = tab[bias.bucket[far < 0 ? 0 : 2 * a.reach]];
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] += v;
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                x[i] += tab[bias.bucket[max(-a.reach, min(a.reach, d0 - 8 * (i >> 2) - (i & 3))) + a.reach]];
            }
          }
        }
        float p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = 32 * qt + acc_row(i, h);
          const float2 st = sStat[row];
          p[i] = ex2(fmaf(x[i], cf, Elem<T>::PSHIFT - st.x));
          if (need_mask) {
            bool see = live && (!a.causal || j < max(p0 + acc_row(i, h) + 1, prefix));
            if (qdoc) see = see && sDoc[row] == kdoc;
            if (!see) p[i] = 0.f;
          }
          x[i] = p[i] == 0.f ? 0.f : p[i] * (dp[i] - st.y);
        }
        if (sc.capped) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= fmaf(-th[i], th[i], 1.f);
        }
        if (sizeof(T) == 2 && Elem<T>::PSHIFT != 0.f) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= ds_mul;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const V8 fp = round8<T>(p + 8 * c), fs = round8<T>(x + 8 * c);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            accv[d] = Elem<T>::mma(col_frag<T, D>(sO, 32 * qt + 16 * c, d, lane), fp, accv[d]);
            acck[d] = Elem<T>::mma(col_frag<T, D>(sQ, 32 * qt + 16 * c, d, lane), fs, acck[d]);
          }
        }
      }
      t = tn;
    }
  }
  if (j >= a.Lk) return;
  const int64_t o = (((int64_t)b * a.Lk + j) * a.Hk + kh) * a.dh;
  const float f_k = a.scale / dscale, f_v = ex2(-Elem<T>::PSHIFT);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dim = 32 * d + 8 * q + 4 * h;
      if (dim < a.dh) {
        typename Elem<T>::V4 vk, vv;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          vk[e] = (T)(live ? acck[d][4 * q + e] * f_k : 0.f);
          vv[e] = (T)(live ? accv[d][4 * q + e] * f_v : 0.f);
        }
        *(typename Elem<T>::V4 *)((T *)g.dk + o + dim) = vk;
        *(typename Elem<T>::V4 *)((T *)g.dv + o + dim) = vv;
      }
    }
}

// The gradient of the learned bias over the tiles within the reach (the dQ kernel has summed the others).  Sums of millions of
// signed terms that have to come out right to fp32: dU is recomputed with the exact delta of each row, and every lane adds into
// a column of its own of a [bucket][lane] array in LDS, so that the order of the additions is the program's.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1) mmt_long_attn_table_kernel(const Args g, float *part) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BK = L::BK, NK = BK / 32, NC = D / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  char *sK = smem, *sV = smem + L::BYTES;
  int *sDoc = (int *)(smem + 2 * L::BYTES), *sB = sDoc + BK;
  BiasLds bias;
  bias.table = (float *)(sB + 6 * WAVES);
  bias.bucket = (unsigned char *)(bias.table + a.n_buckets);
  float *hist = (float *)(bias.bucket + ((2 * a.reach + 1 + 15) & ~15));
  const int item = xcd_item(g.items);
  if (item < 0) return;
  int n = item;
  const int gi = n % g.G;
  n /= g.G;
  const int qt = n % g.nqt;
  n /= g.nqt;
  const int kh = n % a.Hk, b = n / a.Hk, head = kh * g.G + gi;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b);
  const Row w = make_row(g, b, head, qt * ROWS + wave * 32 + col, len);
  const Bounds wb = wave_bounds(w);
  const Bounds gb = group_bounds(wb, sB, wave);
  bias.fill(a, head, 1);
  float *mine = hist + (int64_t)wave * a.n_buckets * 64 + lane;
  for (int k = 0; k < a.n_buckets; ++k) mine[k * 64] = 0.f;
  const int64_t r = ((int64_t)b * a.H + head) * a.Lq + min(w.i, a.Lq - 1);
  const float lse2 = w.live ? g.stat[r].x : INFINITY, delta = w.live ? g.delta_fix[r] : 0.f;
  const T *qrow = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)min(w.i, a.Lq - 1) * a.q_rs + (int64_t)head * a.q_hs;
  const T *drow = (const T *)g.dout + (int64_t)b * g.do_bs + (int64_t)min(w.i, a.Lq - 1) * g.do_rs + (int64_t)head * g.do_hs;
  V8 fq[NC], fd[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    fq[c] = mem_frag<T>(qrow, c, h, a.dh, w.live);
    fd[c] = mem_frag<T>(drow, c, h, a.dh, w.live);
  }
  const ScoreCtx sc = score_ctx(a);
  const int tiles = (gb.hi_max + BK - 1) / BK;
  const DocRange *rng = g.krng ? g.krng + (int64_t)b * g.nkt : nullptr;
  const T *kbase = (const T *)a.k + (int64_t)b * a.k_bs + (int64_t)kh * a.k_hs;
  const T *vbase = (const T *)a.v + (int64_t)b * a.v_bs + (int64_t)kh * a.v_hs;
  const int *kdoc = a.k_doc ? a.k_doc + (int64_t)b * a.Lk : nullptr;
  // tiles with k0 + BK - 1 - p_min > -reach and k0 - p_max < reach
  int t0 = 0, t1 = 0;
  if (gb.hi_max > 0) {
    t0 = max(0, (gb.p_min - a.reach - BK + 1) / BK);
    while (t0 < tiles && t0 * BK + BK - 1 - gb.p_min <= -a.reach) ++t0;
    t1 = min(tiles, max(0, gb.p_max + a.reach + BK) / BK + 1);
    while (t1 > t0 && (t1 - 1) * BK - gb.p_max >= a.reach) --t1;
  }
  Stage<T, D> st;
  for (int t = t0; t < t1; ++t) {
    if (rng && (rng[t].lo > gb.d_max || rng[t].hi < gb.d_min)) continue;
    const int k0 = t * BK;
    __syncthreads();
    st.load(kbase, a.k_rs, k0, a.Lk, a.dh);
    st.store(sK, k0, len, kdoc);
    st.load(vbase, a.v_rs, k0, a.Lk, a.dh);
    st.store(sV, k0, len, kdoc);
    if (kdoc && threadIdx.x < BK) sDoc[threadIdx.x] = k0 + (int)threadIdx.x < a.Lk ? kdoc[k0 + threadIdx.x] : -1;
    __syncthreads();
    if (k0 >= wb.hi_max) continue;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        s = Elem<T>::mma(row_frag<T, D>(sK, 32 * kt + col, c, h), fq[c], s);
        dp = Elem<T>::mma(row_frag<T, D>(sV, 32 * kt + col, c, h), fd[c], dp);
      }
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = s[i];
      const float cf = transform<16, false>(a, sc, x, nullptr, k0 + 32 * kt, h, w.p, w.slope, bias.table, bias.bucket, 0, true, w.hi, w.doc,
                                            kdoc ? sDoc + 32 * kt : nullptr);
      const int d0 = k0 + 32 * kt + 4 * h - w.p;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = ex2(fmaf(x[i], cf, -lse2)), u = p == 0.f ? 0.f : p * (dp[i] - delta);
        const int d = max(-a.reach, min(a.reach, d0 + 8 * (i >> 2) + (i & 3))) + a.reach;
        mine[bias.bucket[d] * 64] += u;
      }
    }
  }
  __syncthreads();
  // columns -> one value per bucket, in a fixed order: wave u takes buckets u, u + 4, ..
  for (int k = wave; k < a.n_buckets; k += WAVES) {
    float v = 0.f;
    for (int u = 0; u < WAVES; ++u) v += hist[((int64_t)u * a.n_buckets + k) * 64 + lane];
    v = wave_sum(v);
    if (lane == 0) part[(((int64_t)b * g.nqt + qt) * a.H + head) * a.n_buckets + k] = v;
  }
}

// the parts of all (batch row, query tile) pairs, in 64 bits and in order; one wave per (head, bucket)
__global__ void mmt_long_attn_table_sum_kernel(const mmt_long_attention a, int64_t n, const float *part, const float *far_part, float *dtable) {
  const int hd = blockIdx.x / a.n_buckets, k = blockIdx.x % a.n_buckets, lane = threadIdx.x;
  const int left = max(0, min(a.rel_buckets[0], a.n_buckets - 1)), right = max(0, min(a.rel_buckets[2 * a.reach], a.n_buckets - 1));
  double v = 0.;
  for (int64_t i = lane; i < n; i += 64) {
    v += part[(i * a.H + hd) * a.n_buckets + k];
    if (k == left) v += far_part[(i * a.H + hd) * 2];
    if (k == right) v += far_part[(i * a.H + hd) * 2 + 1];
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  if (lane == 0) dtable[(int64_t)hd * a.n_buckets + k] = (float)v;
}

// -------------------------------------------------------------------------------------------------------------- host side
static int launch_status(const char *who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MMT_OK : mmt_set_error(MMT_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}

static int elem_size(int dtype) { return dtype == MMT_F32 ? 4 : 2; }
static int tile_keys(int dtype) { return dtype == MMT_F32 ? 32 : 64; }
static int head_tile(int dh) { return dh <= 32 ? 32 : dh <= 64 ? 64 : dh <= 96 ? 96 : 128; }

static int check(const mmt_long_attention *a, const char *who) {
  if (!a || !a->q || !a->k || !a->v) return mmt_set_error(MMT_EINVAL, "%s: null pointer", who);
  if (a->dtype != MMT_F32 && a->dtype != MMT_BF16 && a->dtype != MMT_F16)
    return mmt_set_error(MMT_EINVAL, "%s: unknown element type %d", who, a->dtype);
  if (a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->Lq <= 0 || a->Lk <= 0)
    return mmt_set_error(MMT_EINVAL, "%s: B, H, Hk, Lq and Lk have to be positive", who);
  if (a->H % a->Hk) return mmt_set_error(MMT_EINVAL, "%s: %d query heads are no multiple of %d key heads", who, a->H, a->Hk);
  if (a->dh < 8 || a->dh > 128 || a->dh % 8) return mmt_set_error(MMT_EINVAL, "%s: head size %d, need a multiple of 8 up to 128", who, a->dh);
  if (!(a->scale > 0.f) || !isfinite(a->scale)) return mmt_set_error(MMT_EINVAL, "%s: the scale has to be positive and finite", who);
  if (!(a->softcap >= 0.f) || !isfinite(a->softcap)) return mmt_set_error(MMT_EINVAL, "%s: the cap has to be finite and not negative", who);
  if (a->prefix && !a->causal) return mmt_set_error(MMT_EINVAL, "%s: a prefix is an exception from the causal mask", who);
  if (!a->q_doc != !a->k_doc) return mmt_set_error(MMT_EINVAL, "%s: documents need ids for the queries and the keys", who);
  if (!a->rel_bias != !a->rel_buckets) return mmt_set_error(MMT_EINVAL, "%s: a learned bias needs its table and its buckets", who);
  if (a->rel_bias && (a->n_buckets < 1 || a->n_buckets > 64 || a->reach < 1 || a->reach > 4096))
    return mmt_set_error(MMT_EINVAL, "%s: need 1..64 buckets and a reach of 1..4096", who);
  if (a->rel_bias && (int64_t)(a->H / a->Hk) * a->n_buckets > 8192)
    return mmt_set_error(MMT_EINVAL, "%s: at most 8192 bias entries per key head", who);
  if (a->Lk > (1 << 30) || a->Lq > (1 << 30)) return mmt_set_error(MMT_EINVAL, "%s: at most 2^30 tokens per row", who);
  const int64_t unit = 16 / elem_size(a->dtype);
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) & 15 ||
      (a->q_bs | a->q_rs | a->q_hs | a->k_bs | a->k_rs | a->k_hs | a->v_bs | a->v_rs | a->v_hs) % unit)
    return mmt_set_error(MMT_EINVAL, "%s: rows of q, k and v have to start at multiples of 16 bytes", who);
  const double items = (double)a->B * a->H * (((double)a->Lq + ROWS - 1) / ROWS) + (double)a->B * a->Hk * (((double)a->Lk + ROWS - 1) / ROWS);
  if (items > 3e7 || (double)a->B * a->H * a->Lq > 2e9) return mmt_set_error(MMT_EINVAL, "%s: too many rows for one call", who);
  return MMT_OK;
}

// Splits of the keys (forward): enough workgroups for two on each of the 256 CUs, at least four tiles each
static void plan(Args &g) {
  const mmt_long_attention &a = g.a;
  const int bk = tile_keys(a.dtype);
  g.G = a.H / a.Hk;
  // few queries: the rows of all heads that share a key head go into one tile, which reads the cache once
  g.pack = g.G > 1 && (int64_t)a.Lq * g.G <= ROWS ? g.G : 1;
  g.nqt = (int)(((int64_t)a.Lq * g.pack + ROWS - 1) / ROWS);
  g.nkt = (a.Lk + bk - 1) / bk;
  const int64_t base = (int64_t)a.B * a.Hk * (g.pack > 1 ? 1 : g.G) * g.nqt;
  g.nsplit = 1;
  if (base < 256) g.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>((512 + base - 1) / base, g.nkt / 4));
  g.items = (int)(base * g.nsplit);
}

static size_t align64(size_t n) { return (n + 63) & ~(size_t)63; }
static size_t doc_bytes(const mmt_long_attention &a) {
  if (!a.q_doc) return 0;
  const size_t bk = tile_keys(a.dtype);
  return align64(sizeof(DocRange) * a.B * ((a.Lk + bk - 1) / bk)) + align64(sizeof(DocRange) * a.B * ((a.Lq + bk - 1) / bk));
}

static dim3 grid8(int items) { return dim3(8 * ((items + 7) / 8)); }

static char *doc_ranges(Args &g, char *ws, bool queries, hipStream_t st) {
  const mmt_long_attention &a = g.a;
  if (!a.q_doc) return ws;
  const int bk = tile_keys(a.dtype);
  const int nk = a.B * g.nkt, nqb = (a.Lq + bk - 1) / bk, nq = a.B * nqb;
  DocRange *k = (DocRange *)ws, *q = (DocRange *)(ws + align64(sizeof(DocRange) * nk));
  hipLaunchKernelGGL(mmt_long_attn_docs_kernel, dim3((nk + 3) / 4), dim3(256), 0, st, a.k_doc, a.Lk, g.nkt, bk, nk, k);
  if (queries) hipLaunchKernelGGL(mmt_long_attn_docs_kernel, dim3((nq + 3) / 4), dim3(256), 0, st, a.q_doc, a.Lq, nqb, bk, nq, q);
  g.krng = k, g.qrng = q;
  return ws + doc_bytes(a);
}

template <typename K> static void launch(K kernel, dim3 grid, size_t lds, hipStream_t st, const Args &g) {
  (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL(kernel, grid, dim3(THREADS), lds, st, g);
}

template <typename T, int D> static void run_fwd(const Args &g, hipStream_t st) {
  const size_t lds = 2 * Tile<T, D>::BYTES + 4 * Tile<T, D>::BK + 24 * WAVES + bias_lds_bytes(g.a, g.pack);
  launch(mmt_long_attn_fwd_kernel<T, D>, grid8(g.items), lds, st, g);
  if (g.nsplit > 1) {
    const int64_t rows = (int64_t)g.a.B * g.a.H * g.a.Lq;
    hipLaunchKernelGGL(mmt_long_attn_join_kernel<T>, dim3((rows + 15) / 16), dim3(256), 0, st, g);
  }
}

template <typename T, int D> static void run_bwd(Args &g, hipStream_t st, float *table_part, float *dtable) {
  const mmt_long_attention &a = g.a;
  const size_t tiles = 2 * Tile<T, D>::BYTES + 4 * Tile<T, D>::BK + 24 * WAVES;
  g.items = a.B * a.H * g.nqt;
  launch(mmt_long_attn_dq_kernel<T, D>, grid8(g.items), tiles + bias_lds_bytes(a, 1), st, g);
  if (a.rel_bias) {
    const size_t lds = tiles + bias_lds_bytes(a, 1) + (size_t)WAVES * a.n_buckets * 256;
    (void)hipFuncSetAttribute((const void *)mmt_long_attn_table_kernel<T, D>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL((mmt_long_attn_table_kernel<T, D>), grid8(g.items), dim3(THREADS), lds, st, g, table_part);
    hipLaunchKernelGGL(mmt_long_attn_table_sum_kernel, dim3(a.H * a.n_buckets), dim3(64), 0, st, a, (int64_t)a.B * g.nqt, table_part,
                       g.far_part, dtable);
  }
  g.items = a.B * a.Hk * ((a.Lk + ROWS - 1) / ROWS);
  launch(mmt_long_attn_dkv_kernel<T, D>, grid8(g.items), tiles + 8 * Tile<T, D>::BK + bias_lds_bytes(a, g.G), st, g);
}

#define LA_DISPATCH(dtype, dh, CALL)                                   \
  do {                                                                 \
    const int d_ = head_tile(dh);                                      \
    if ((dtype) == MMT_BF16) { typedef __bf16 T; LA_HEADS(T, CALL) }   \
    else if ((dtype) == MMT_F16) { typedef _Float16 T; LA_HEADS(T, CALL) } \
    else { typedef float T; LA_HEADS(T, CALL) }                        \
  } while (0)
#define LA_HEADS(T, CALL)                 \
  if (d_ == 32) { CALL(T, 32); }          \
  else if (d_ == 64) { CALL(T, 64); }     \
  else if (d_ == 96) { CALL(T, 96); }     \
  else { CALL(T, 128); }

struct Workspace {                 // one piece after another, each a multiple of 64 bytes
  size_t docs, part_o, part_ml, stat, fix, far, table, maxima, total;
};
static Workspace layout(const Args &g, bool backward) {
  const mmt_long_attention &a = g.a;
  Workspace w = {};
  const size_t rows = (size_t)a.B * a.H * a.Lq, tiles = (size_t)a.B * ((a.Lq + ROWS - 1) / ROWS) * a.H;
  size_t n = 0;
  w.docs = n, n += doc_bytes(a);
  if (!backward) {
    if (g.nsplit > 1) {
      w.part_o = n, n += align64(4 * rows * a.dh * g.nsplit);
      w.part_ml = n, n += align64(8 * rows * g.nsplit);
    }
  } else {
    w.stat = n, n += align64(8 * rows);
    w.maxima = n, n += 64;
    if (a.rel_bias) {
      w.fix = n, n += align64(4 * rows);
      w.far = n, n += align64(8 * tiles);
      w.table = n, n += align64(4 * tiles * a.n_buckets);
    }
  }
  w.total = n;
  return w;
}

}  // namespace la

using namespace la;

extern "C" size_t mmt_long_attention_workspace_bytes(const mmt_long_attention *a, int backward) {
  if (check(a, "mmt_long_attention_workspace_bytes")) return 0;
  Args g = {};
  g.a = *a;
  plan(g);
  return layout(g, backward != 0).total;
}

extern "C" int mmt_long_attention_fwd(const mmt_long_attention *a, void *out, float *lse, void *workspace, size_t workspace_bytes,
                                      void *stream) {
  if (int rc = check(a, "mmt_long_attention_fwd")) return rc;
  if (!out || (uintptr_t)out & 15) return mmt_set_error(MMT_EINVAL, "mmt_long_attention_fwd: out has to be a 16-byte aligned address");
  Args g = {};
  g.a = *a;
  plan(g);
  const Workspace w = layout(g, false);
  if (w.total && (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < w.total))
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_fwd: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, w.total);
  hipStream_t st = (hipStream_t)stream;
  char *ws = (char *)workspace;
  g.out = out, g.lse = lse;
  g.part_o = (float *)(ws + w.part_o), g.part_ml = (float *)(ws + w.part_ml);
  doc_ranges(g, ws + w.docs, false, st);
#define CALL(T, D) run_fwd<T, D>(g, st)
  LA_DISPATCH(a->dtype, a->dh, CALL);
#undef CALL
  return launch_status("mmt_long_attention_fwd");
}

extern "C" int mmt_long_attention_bwd(const mmt_long_attention *a, const void *out, const float *lse, const void *dout, int64_t do_bs,
                                      int64_t do_rs, int64_t do_hs, const float *dlse, void *dq, void *dk, void *dv, float *drel_bias,
                                      void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = check(a, "mmt_long_attention_bwd")) return rc;
  if (!out || !lse || !dout || !dq || !dk || !dv || (a->rel_bias && !drel_bias))
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_bwd: null pointer");
  if (((uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15 ||
      (do_bs | do_rs | do_hs) % (16 / elem_size(a->dtype)))
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_bwd: rows have to start at multiples of 16 bytes");
  Args g = {};
  g.a = *a;
  plan(g);
  g.pack = 1, g.nsplit = 1, g.nqt = (a->Lq + ROWS - 1) / ROWS;
  const Workspace w = layout(g, true);
  if (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < w.total)
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_bwd: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, w.total);
  hipStream_t st = (hipStream_t)stream;
  char *ws = (char *)workspace;
  g.out = const_cast<void *>(out), g.lse = const_cast<float *>(lse);
  g.dout = dout, g.do_bs = do_bs, g.do_rs = do_rs, g.do_hs = do_hs;
  g.dq = dq, g.dk = dk, g.dv = dv, g.dlse = dlse;
  g.stat = (const float2 *)(ws + w.stat);
  if (a->rel_bias) g.delta_fix = (float *)(ws + w.fix), g.far_part = (float *)(ws + w.far);
  doc_ranges(g, ws + w.docs, true, st);
  unsigned *maxima = nullptr;
  if (a->dtype == MMT_F16) {
    maxima = (unsigned *)(ws + w.maxima);
    g.dscale = (const float *)(maxima + 4);
    hipLaunchKernelGGL(mmt_long_attn_zero_kernel, dim3(1), dim3(64), 0, st, maxima, 8);
    const int64_t rows = (int64_t)a->B * a->Lk * a->Hk;
    hipLaunchKernelGGL(mmt_long_attn_vnorm_kernel<_Float16>, dim3((unsigned)std::min<int64_t>((rows + 15) / 16, 2048)), dim3(256), 0, st, g, maxima);
  }
  const int64_t rows = (int64_t)a->B * a->Lq * a->H;
  const dim3 grid((unsigned)std::min<int64_t>((rows + 15) / 16, 8192));
  float2 *stat = (float2 *)(ws + w.stat);
  if (a->dtype == MMT_BF16) hipLaunchKernelGGL(mmt_long_attn_stat_kernel<__bf16>, grid, dim3(256), 0, st, g, dlse, stat, maxima);
  else if (a->dtype == MMT_F16) hipLaunchKernelGGL(mmt_long_attn_stat_kernel<_Float16>, grid, dim3(256), 0, st, g, dlse, stat, maxima);
  else hipLaunchKernelGGL(mmt_long_attn_stat_kernel<float>, grid, dim3(256), 0, st, g, dlse, stat, maxima);
  if (maxima) hipLaunchKernelGGL(mmt_long_attn_dscale_kernel, dim3(1), dim3(1), 0, st, maxima, (float *)(maxima + 4));
#define CALL(T, D) run_bwd<T, D>(g, st, (float *)(ws + w.table), drel_bias)
  LA_DISPATCH(a->dtype, a->dh, CALL);
#undef CALL
  return launch_status("mmt_long_attention_bwd");
}
