// The kernels of attention over long rows and their launchers, included by one translation unit per element type
// (long_attention_{bf16,fp16,fp32}.hip); the entry points are in long_attention.hip.
#pragma once
#include "long_attention.cuh"
#include "long_attention_args.cuh"

namespace la {

// what a lane knows about its query row
struct Row {
  bool valid, live;                // a row of this call; and not padding
  int i, h, p, hi, doc;            // query, head, position, first invisible key (before documents), document
  float slope;                     // slope times log2 e
};

template <typename A> __device__ __forceinline__ int row_len(const A &a, int b) {
  return a.kv_len ? max(0, min(scalar_load(a.kv_len + b), a.Lk)) : a.Lk;
}

// first invisible key of position p, before documents
__device__ __forceinline__ int visible_end(const mmt_long_attention &a, int len, int prefix, int p) {
  return a.causal ? min(len, max(p + 1, prefix)) : len;
}
// (the document and the slope are only on their way: dead rows, and settle(slope), where they are needed)
__device__ __forceinline__ Row make_row(const Args &g, int b, int head0, int r, int len, int prefix) {
  const mmt_long_attention &a = g.a;
  Row w;
  w.i = r / g.pack;
  w.h = head0 + r % g.pack;
  w.valid = w.i < a.Lq;
  w.p = len - a.Lq + w.i;
  w.doc = 0;
  if (a.q_doc) w.doc = a.q_doc[(int64_t)b * a.Lq + min(w.i, a.Lq - 1)];
  w.slope = a.slopes ? a.slopes[w.h] * LOG2E : 0.f;
  w.live = w.valid && w.doc >= 0;
  w.hi = visible_end(a, len, prefix, w.p);
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
// without documents they follow from the first and the last of rows r0 .. r0 + n - 1
__device__ __forceinline__ Bounds range_bounds(const Args &g, int r0, int n, int len, int prefix) {
  const mmt_long_attention &a = g.a;
  const int i0 = r0 / g.pack, i1 = min(a.Lq - 1, (r0 + n - 1) / g.pack), off = len - a.Lq;
  if (i0 > i1) return Bounds{0x7fffffff, 0, 0x7fffffff, -0x7fffffff, 0x7fffffff, -1};
  return Bounds{visible_end(a, len, prefix, off + i0), max(0, visible_end(a, len, prefix, off + i1)), off + i0, off + i1, 0, 0};
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

// The learned bias in LDS, in units of log 2.  Bucket numbers outside the table are clamped into it.  Entries count as clamped to
// -2^14 .. 2^14: next to another visible key e^-2^14 is 0 all the same, and of a row all of whose keys carry a mask's constant such as
// -1e9 fp32 would keep no digit of the scores, nor the log-sum enough to form the probabilities again (gradients 20 times too large at
// -1e9, 2 % off at -1e6).  At or below -2^100 (-inf, the lowest value of fp32 and bf16) an entry hides its bucket like a mask.
__device__ __forceinline__ float bias_entry(const mmt_long_attention &a, int head, int bucket) {
  const float v = a.rel_bias[(int64_t)head * a.n_buckets + bucket];
  return (v <= -0x1p100f ? -INFINITY : v < -0x1p14f ? -0x1p14f : v > 0x1p14f ? 0x1p14f : v) * LOG2E;      // (NaN stays)
}
__device__ __forceinline__ int bias_bucket(const mmt_long_attention &a, int d) {
  return max(0, min(a.rel_buckets[max(-a.reach, min(a.reach, d)) + a.reach], a.n_buckets - 1));
}
// One head: the bias of every distance from -reach - PAD to reach + PAD, so that a tile that is not wholly beyond the reach finds all
// of its distances (128 rows x 64 keys span 190) at constant steps from one address.
constexpr int PAD = 192;
struct Lut {
  float *mid;                      // of distance 0
  static __host__ __device__ int floats(const mmt_long_attention &a) { return a.rel_bias ? (2 * (a.reach + PAD) + 4) & ~3 : 0; }
  // `bucket` (of distance 0), where it is wanted, receives the bucket numbers too.  Every wave holds the table, one entry per lane, and
  // asks for the buckets of several distances at once: two waits for memory, whatever the reach.
  template <int THREADS_ = THREADS> __device__ __forceinline__ void fill(const mmt_long_attention &a, int head, unsigned char *bucket = nullptr) const {
    constexpr int AT_ONCE = 1024 / THREADS_;
    const float entry = bias_entry(a, head, min((int)(threadIdx.x & 63), a.n_buckets - 1));
    const int first = -a.reach - PAD, last = a.reach + PAD;
    for (int d0 = first; d0 <= last; d0 += 1024) {
      int k[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) k[u] = bias_bucket(a, d0 + u * THREADS_ + (int)threadIdx.x);
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int d = d0 + u * THREADS_ + (int)threadIdx.x;
        const float v = __shfl(entry, k[u]);
        if (d > last) continue;
        mid[d] = v;
        if (bucket) bucket[d] = (unsigned char)k[u];
      }
    }
  }
};
// Several heads (few queries): their table rows, and the bucket of each clamped distance
struct PackedBias {
  float *table;                    // [pack][n_buckets]
  unsigned char *bucket;           // [2 reach + 1]
  static __host__ __device__ int bytes(const mmt_long_attention &a, int pack) {
    return a.rel_bias ? pack * a.n_buckets * 4 + ((2 * a.reach + 1 + 15) & ~15) : 0;
  }
  __device__ __forceinline__ void fill(const mmt_long_attention &a, int head0, int pack) {
    for (int n = threadIdx.x; n < pack * a.n_buckets; n += blockDim.x) table[n] = bias_entry(a, head0 + n / a.n_buckets, n % a.n_buckets);
    for (int n = threadIdx.x; n < 2 * a.reach + 1; n += blockDim.x) bucket[n] = (unsigned char)bias_bucket(a, n - a.reach);
  }
};

// Raw products -> modified scores in units of log 2; `t` receives tanh(s / cap) when the scores are capped and the caller needs it.
struct ScoreCtx {
  float c_scale, cap_in, cap_out;  // scale log2 e; scale / cap; cap log2 e
  bool capped, rel, sloped;
};
__device__ __forceinline__ ScoreCtx score_ctx(const mmt_long_attention &a) {
  ScoreCtx s;
  s.c_scale = a.scale * LOG2E;
  s.capped = a.softcap > 0.f;
  s.cap_in = s.capped ? a.scale / a.softcap : 0.f;
  s.cap_out = a.softcap * LOG2E;
  s.rel = a.rel_bias != nullptr;
  s.sloped = a.slopes != nullptr;
  return s;
}
// where a tile lies: d_lo .. d_hi is the range of its distances over the wave's rows
struct Place {
  int far;                         // wholly beyond the reach: -1 behind, 1 ahead; 0 within it
  int side;                        // distances of one sign: -1 none positive, 1 none negative; 0 both
};
__device__ __forceinline__ Place place(const mmt_long_attention &a, int d_lo, int d_hi) {
  Place p;
  p.far = d_hi <= -a.reach ? -1 : d_lo >= a.reach ? 1 : 0;
  p.side = d_hi <= 0 ? -1 : d_lo >= 0 ? 1 : 0;
  return p;
}
// x: 16 raw products of a lane, element i belongs to the distance d0 + STEP (8 (i / 4) + i % 4), STEP 1 or -1.
// One multiplication and addition takes up the scale, the bias of a tile beyond the reach and, with distances of one sign, the lane's
// part of the slope; what is left of the slope is a constant per element.  Where nothing else is left the scores stay as they are and
// the multiplication and addition are returned, for the one in front of the exponential.
struct Linear {
  float mul, add;                  // score = x mul + add, mul > 0
};
template <int STEP, bool KEEP, bool PACKED>
__device__ __forceinline__ Linear modify(const mmt_long_attention &a, const ScoreCtx &sc, float *x, float *t, int d0, float slope, const float *lut,
                                       const unsigned char *bucket, Place at) {
  float mul = sc.c_scale, add = 0.f;
  if (sc.capped) {
    tanh_scores<16>(x, sc.cap_in);
    if (KEEP) {
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = x[i];
    }
    mul = sc.cap_out;
  }
  if (sc.rel && at.far != 0) add = PACKED ? lut[bucket[at.far < 0 ? 0 : 2 * a.reach]] : lut[at.far < 0 ? -a.reach : a.reach];
  const float s1 = at.side < 0 ? slope : -slope;          // u += s1 * distance
  if (!sc.sloped && !(sc.rel && at.far == 0)) return Linear{mul, add};
  if (sc.sloped && at.side != 0) add = fmaf(s1, (float)d0, add);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = fmaf(x[i], mul, add);
  if (sc.sloped) {
    if (at.side != 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = fmaf(s1, (float)(STEP * (8 * (i >> 2) + (i & 3))), x[i]);
    } else {
      const float f0 = (float)d0;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = fmaf(-slope, fabsf(f0 + (float)(STEP * (8 * (i >> 2) + (i & 3)))), x[i]);
    }
  }
  if (sc.rel && at.far == 0) {
    if constexpr (PACKED) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] += lut[bucket[max(-a.reach, min(a.reach, d0 + STEP * (8 * (i >> 2) + (i & 3)))) + a.reach]];
    } else {
      // (rows that are not live may stand anywhere: their address is held inside the table)
      const int lo = max(-a.reach - PAD, min(a.reach + PAD - 27, STEP > 0 ? d0 : d0 - 27));
      const float *p = lut + lo;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = 8 * (i >> 2) + (i & 3);
        x[i] += p[STEP > 0 ? e : 27 - e];
      }
    }
  }
  return Linear{1.f, 0.f};
}
// what a row does not see -> -inf; key j of the sub-tile is the accumulator's row
__device__ __forceinline__ void mask_keys(float *x, int key0, int hi, const int *sDoc, int doc, int h) {
  asm volatile("" : "+v"(h));                             // (few tiles: see rare_tid)
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = key0 + acc_row(i, h) < hi ? x[i] : -INFINITY;
  if (sDoc) {
    int id[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) id[i] = sDoc[acc_row(i, h)];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = id[i] == doc ? x[i] : -INFINITY;
  }
}

// ---------------------------------------------------------------------------------------------------------------- forward
// One wave's 32 rows against NK x 32 keys of a tile in LDS: products, modification, masks, running maximum and sum, o^T += v^T P^T.
// The running maximum (FwdState::m, or up to SLACK less than it) is in units of log 2.
template <typename T, int D> struct FwdState {
  f32x16 acc[D / 32];
  float m, l;
};
template <typename T, int D, bool GAPS, int NK>
__device__ __forceinline__ void fwd_products(float *x, const typename Elem<T>::V8 *fq, const char *sK, int lane, int dh) {
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) {
    f32x16 s = {};
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      if (has_chunk<GAPS, D / 16>(c, dh)) s = Elem<T>::mma(row_frag<T, D>(sK, 32 * kt + (lane & 31), c, lane >> 5), fq[c], s);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[16 * kt + i] = s[i];
  }
}
// products -> probabilities (not yet divided by their sum)
template <typename T, int D, bool MOD, bool PACKED, int NK>
__device__ __forceinline__ void fwd_softmax(FwdState<T, D> &st, float *x, int key0, const Row &w, const mmt_long_attention &a, const ScoreCtx &sc,
                                            const float *lut, const unsigned char *bucket, Place at, bool need_mask, const int *sDoc, int h) {
  constexpr int ND = D / 32;
  Linear f = {sc.c_scale, 0.f};
  if constexpr (MOD) {
    static_assert(NK == 1, "modified scores come 32 keys at a time");
    f = modify<1, false, PACKED>(a, sc, x, nullptr, key0 + 4 * h - w.p, w.slope, lut, bucket, at);
  }
  if (need_mask) {
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) mask_keys(x + 16 * kt, key0 + 32 * kt, w.hi, sDoc ? sDoc + 32 * kt : nullptr, w.doc, h);
  }
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < NK * 16; ++i) mx = fmaxf(mx, x[i]);
  // What the exponentials refer to follows the maximum only where that has gone SLACK ahead: sums and accumulators are rescaled in the
  // first tiles of a row, not in every one that raises the maximum of one of 32 rows.
  const float m_new = fmaxf(st.m, fmaf(half_max(mx), f.mul, f.add));
  const bool moved = m_new - st.m > Elem<T>::SLACK;
  const float ref = moved ? m_new : st.m, ms = ref == -INFINITY ? 0.f : ref;
  const float alpha = moved ? ex2(st.m - ms) : 1.f;
  st.m = ref;
  const float off = Elem<T>::PSHIFT + (f.add - ms);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NK * 16; ++i) {
    x[i] = ex2(fmaf(x[i], f.mul, off));
    sum += x[i];
  }
  st.l = fmaf(st.l, alpha, sum);
  if (__any(moved)) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.acc[d][i] *= alpha;
  }
}
template <typename T, int D, int NK> __device__ __forceinline__ void fwd_values(FwdState<T, D> &st, const float *x, const char *sV, int lane) {
  constexpr int ND = D / 32;
#pragma unroll
  for (int c = 0; c < NK * 2; ++c) {
    const typename Elem<T>::V8 p = round8<T>(x + 8 * c);
#pragma unroll
    for (int d = 0; d < ND; ++d) st.acc[d] = Elem<T>::mma(col_frag<T, D>(sV, 16 * c, d, lane), p, st.acc[d]);
  }
}

// A row's result: o^T of the accumulator scaled, or this split's part of it
template <typename T, int D>
__device__ __forceinline__ void fwd_store(const Args &g, const FwdState<T, D> &st, const Row &w, int b, int split, int h) {
  constexpr int ND = D / 32;
  const mmt_long_attention &a = g.a;
  const float l = half_sum(st.l);
  if (!w.valid) return;
  const int64_t r = ((int64_t)b * a.H + w.h) * a.Lq + w.i;
  if (g.nsplit > 1) {
    const int64_t rs = (int64_t)split * a.B * a.H * a.Lq + r;
    if (h == 0) {
      g.part_ml[2 * rs] = w.live ? st.m : -INFINITY;
      g.part_ml[2 * rs + 1] = w.live ? l : 0.f;
    }
    float *o = g.part_o + rs * a.dh;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int dim = 32 * d + 8 * q + 4 * h;
        if (dim < a.dh) *(f32x4 *)(o + dim) = f32x4{st.acc[d][4 * q], st.acc[d][4 * q + 1], st.acc[d][4 * q + 2], st.acc[d][4 * q + 3]};
      }
    return;
  }
  const bool some = w.live && l != 0.f;                   // (a NaN sum is "some")
  const float inv = some ? 1.f / l : 0.f;
  if (g.lse && h == 0) g.lse[r] = some ? (st.m + log2f(l * ex2(-Elem<T>::PSHIFT))) * LN2 : -INFINITY;
  const int64_t o = (((int64_t)b * a.Lq + w.i) * a.H + w.h) * a.dh;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dim = 32 * d + 8 * q + 4 * h;
      if (dim < a.dh) {
        typename Elem<T>::V4 v, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = some ? st.acc[d][4 * q + e] * inv : 0.f;
          v[e] = (T)y, lo[e] = (T)(y - (float)v[e]);
        }
        *(typename Elem<T>::V4 *)((T *)g.out + o + dim) = v;
        if (g.low) *(typename Elem<T>::V4 *)((T *)g.low + o + dim) = lo;
      }
    }
}

// One workgroup = 128 rows (4 waves x 32) of one head - or, without a learned bias and where that takes fewer tiles, of all heads that
// share a key head - against a range of key tiles.  K and V tiles go straight from memory to LDS, one
// tile ahead of the products (two buffers, one barrier per tile).  MOD: the scores are capped or biased; without it they go from the
// product into the exponential as they are.
// S is computed transposed (the accumulator's rows are keys, its columns the wave's queries), so that a lane owns one query: maximum and
// sum need one exchange between the two lane halves, and the rounded P is already the operand of the second product.
// Measured, bf16 causal 8192 tokens x 16 heads of 128 over 4, learned bias: 319 us, 860 TFLOP/s of the 1156 that a large library product
// reaches; non-causal 2 x 2048 x 16 heads of 64: 61 us, 570; unmodified, causal 2 x 4096 x 16 heads of 128 over 4: 159 us, 860.  Bound by the vector instructions of the softmax (48 and 55 % of the cycles)
// between the matrix instructions (40 and 24 %) at the two waves per SIMD that the registers allow; LDS is at 32 and 21 %, without bank
// conflicts.
// TEAMS = 2: eight waves, two per 32 rows, which deal the key tiles among themselves and join at the end (rule and figures at teams()).
template <typename T, int D, bool GAPS, bool MOD, int TEAMS>
__global__ void __launch_bounds__(TEAMS * THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_fwd_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BK = L::BK, NC = D / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  int *sDoc2 = (int *)(smem + TEAMS * 4 * L::BYTES), *sB = sDoc2 + TEAMS * 2 * BK;
  const Lut lut = {(float *)(sB + 6 * WAVES) + a.reach + PAD};
  const int grp = blockIdx.x % g.groups;
  int n = blockIdx.x / g.groups;
  const int split = n % g.nsplit;
  n /= g.nsplit;
  const int ngroup = g.G / g.pack, gi = n % ngroup;
  int qt = n / ngroup;
  if (a.causal) qt = g.nqt - 1 - qt;                     // the tiles with the most keys first
  const int kh = grp % a.Hk, b = grp / a.Hk;
  const int head0 = kh * g.G + gi;
  const int lane = threadIdx.x & 63, w_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = w_all % WAVES, team = w_all / WAVES, h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b), prefix = a.prefix ? scalar_load(a.prefix + b) : 0;
  // what does not depend on one another is requested before any of it is waited for: the time of a short row is these waits
  Row w = make_row(g, b, head0, qt * ROWS + wave * 32 + col, len, prefix);
  const T *qrow = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)min(w.i, a.Lq - 1) * a.q_rs + (int64_t)w.h * a.q_hs;
  V8 fq[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) fq[c] = mem_frag<T>(qrow, c, h, a.dh);
  const DocRange *rng = g.krng ? g.krng + (int64_t)b * g.nkt : nullptr;
  const int *kdoc = a.k_doc ? a.k_doc + (int64_t)b * a.Lk : nullptr;
  DocRange ready = TileIter::ahead(rng, 0, g.nkt);
  Bounds wb, gb;
  if (rng) wb = wave_bounds(w), gb = group_bounds(wb, sB, wave);
  else wb = range_bounds(g, qt * ROWS + wave * 32, 32, len, prefix), gb = range_bounds(g, qt * ROWS, ROWS, len, prefix);
  const int tiles = (gb.hi_max + BK - 1) / BK, per = (tiles + g.nsplit - 1) / g.nsplit;
  if (split) ready = TileIter::ahead(rng, split * per, g.nkt);
  Deal<TEAMS> deal;
  deal.it.start(rng, gb.d_min, gb.d_max, split * per, min(tiles, (split + 1) * per), ready);
  Dma<T, D> dk, dv;
  dk.init((const T *)a.k + (int64_t)b * a.k_bs + (int64_t)kh * a.k_hs, a.k_rs, a.Lk, a.dh);
  dv.init((const T *)a.v + (int64_t)b * a.v_bs + (int64_t)kh * a.v_hs, a.v_rs, a.Lk, a.dh);
  char *const tiles_at = smem + team * 4 * L::BYTES;
  const unsigned lds = lds_address(tiles_at);
  deal.next(team, BK, len);
  int ids = 0;                                           // the document of the tile's key `lane`
  if (deal.t >= 0) {
    dk.load(lds, deal.t * BK);
    dv.load(lds + L::BYTES, deal.t * BK);
    if (kdoc) ids = kdoc[min(deal.t * BK + lane, a.Lk - 1)];
  }
  if (MOD && a.rel_bias) lut.fill<TEAMS * THREADS>(a, head0);
  FwdState<T, D> st;
#pragma unroll
  for (int d = 0; d < D / 32; ++d) st.acc[d] = f32x16{};
  st.m = -INFINITY, st.l = 0.f;
  const ScoreCtx sc = score_ctx(a);
#pragma unroll
  for (int c = 0; c < NC; ++c) live_frag(fq[c], c, h, a.dh, w.live);
  settle(w.slope), settle(w.doc);
  deal.it.here();
  // (the buffer is a constant of the step: every LDS address of the loop is one register and an immediate)
  auto step = [&](auto buffer) {
    constexpr int buf = decltype(buffer)::value;
    const int k0 = deal.t * BK;
    const bool mine = TEAMS == 1 || deal.t >= 0, mixed = deal.mixed, zero = deal.zero, any_zero = deal.any_zero;
    char *sK = tiles_at + buf * 2 * L::BYTES, *sV = sK + L::BYTES;
    int *sDoc = sDoc2 + (TEAMS == 1 ? buf : team * 2 + buf) * BK;
    if (kdoc && wave == 0 && lane < BK) sDoc[lane] = ids;
    dma_wait<0>();
    if constexpr (GAPS) dk.clear_pads(sK, a.dh);
    __syncthreads();                                     // the tile is here, and nobody reads the other buffer any more
    if (any_zero) {                                      // (a key row only reaches scores that are masked: V alone)
      if (zero) zero_rows<T, D>(sV, len - k0, mixed ? sDoc : nullptr);
      __syncthreads();
    }
    deal.next(team, BK, len);
    if (deal.t >= 0) {
      dk.load(lds + (buf ^ 1) * 2 * L::BYTES, deal.t * BK);
      dv.load(lds + (buf ^ 1) * 2 * L::BYTES + L::BYTES, deal.t * BK);
      if (kdoc) ids = kdoc[min(deal.t * BK + lane, a.Lk - 1)];
    }
    if (mine && k0 < wb.hi_max) {
      const bool need_mask = k0 + BK > wb.hi_min || mixed;
      const Place at = place(a, k0 - wb.p_max, k0 + BK - 1 - wb.p_min);
      // modified scores: 32 keys at a time (the modification needs the registers); else all of the tile
      constexpr int NK = MOD ? 1 : BK / 32;
#pragma unroll
      for (int kt = 0; kt < BK / 32; kt += NK) {
        float x[NK * 16];
        fwd_products<T, D, GAPS, NK>(x, fq, sK + kt * 32 * L::NS * 16, lane, a.dh);
        fwd_softmax<T, D, MOD, false, NK>(st, x, k0 + 32 * kt, w, a, sc, lut.mid, nullptr, at, need_mask, mixed ? sDoc + 32 * kt : nullptr, h);
        fwd_values<T, D, NK>(st, x, sV + kt * 32 * L::NS * 16, lane);
      }
    }
    };
  while (deal.lead >= 0) {
    step(Const<0>());
    if (deal.lead < 0) break;
    step(Const<1>());
  }
  if constexpr (TEAMS == 2) {                             // the second team's part of every row, through LDS (the tiles are done with)
    float *s = (float *)smem + threadIdx.x % THREADS;
    __syncthreads();
    if (team) {
      s[0] = st.m, s[THREADS] = st.l;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[(2 + 16 * d + i) * THREADS] = st.acc[d][i];
    }
    __syncthreads();
    if (team) return;
    const float m = fmaxf(st.m, s[0]), ms = m == -INFINITY ? 0.f : m, f0 = ex2(st.m - ms), f1 = ex2(s[0] - ms);
    st.m = m, st.l = fmaf(st.l, f0, s[THREADS] * f1);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.acc[d][i] = fmaf(st.acc[d][i], f0, s[(2 + 16 * d + i) * THREADS] * f1);
  }
  fwd_store(g, st, w, b, split, h);
}

// Few queries (all rows that share a key head fit into 32): the rows are the same for all four waves, which deal the keys among
// themselves, 32 at a time, and meet at the end, where their maxima, sums and accumulators are joined.  Each has one buffer for K and
// one for V: the next keys are requested as soon as the products have been taken from the buffer, the next values after theirs, so
// that 16 KiB per wave at a head size of 128 and, with two workgroups, 128 KiB per CU are on their way.  Bound by reading the cache: 16
// requests of up to 32768 tokens (1.36 GB) x 8 key heads of 128 in bf16 take 285 us, 4.8 TB/s where a copy reaches 4.9 (the
// general kernel: 914 us, three of its four waves without rows).  At a head size of 128 all 256 registers are taken and 48 bytes per lane
// live in scratch.
template <typename T, int D, bool MOD>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_few_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BK = 32, NC = D / 16, ND = D / 32, TILE = BK * L::NS * 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  int *sDocs = (int *)(smem + 2 * WAVES * TILE);
  PackedBias bias;
  bias.table = (float *)(sDocs + BK * WAVES);
  bias.bucket = (unsigned char *)(bias.table + (MOD && a.rel_bias ? g.pack * a.n_buckets : 0));
  const int grp = blockIdx.x % g.groups, split = blockIdx.x / g.groups, kh = grp % a.Hk, b = grp / a.Hk, head0 = kh * g.G;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b), prefix = a.prefix ? scalar_load(a.prefix + b) : 0;
  Row w = make_row(g, b, head0, col, len, prefix);
  const T *qrow = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)min(w.i, a.Lq - 1) * a.q_rs + (int64_t)w.h * a.q_hs;
  V8 fq[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) fq[c] = mem_frag<T>(qrow, c, h, a.dh);
  const Bounds wb = a.q_doc ? wave_bounds(w) : range_bounds(g, 0, 32, len, prefix);
  const int tiles = (wb.hi_max + BK - 1) / BK, workers = g.nsplit * WAVES;
  const int *kdoc = a.k_doc ? a.k_doc + (int64_t)b * a.Lk : nullptr;
  Dma<T, D, BK, 64> dk, dv;
  dk.init((const T *)a.k + (int64_t)b * a.k_bs + (int64_t)kh * a.k_hs, a.k_rs, a.Lk, a.dh);
  dv.init((const T *)a.v + (int64_t)b * a.v_bs + (int64_t)kh * a.v_hs, a.v_rs, a.Lk, a.dh);
  char *sK = smem + wave * 2 * TILE, *sV = sK + TILE;
  int *sDoc = sDocs + wave * BK;
  const unsigned lds = lds_address(sK);
  int t = split * WAVES + wave;                           // neighbouring tiles go to neighbouring waves
  if (t < tiles) {
    dk.load(lds, t * BK);
    dv.load(lds + TILE, t * BK);
  }
  if (MOD && a.rel_bias) {
    bias.fill(a, head0, g.pack);
    __syncthreads();
  }
  const float *tab = bias.table + (w.valid ? w.h - head0 : 0) * a.n_buckets;
  FwdState<T, D> st;
#pragma unroll
  for (int d = 0; d < ND; ++d) st.acc[d] = f32x16{};
  st.m = -INFINITY, st.l = 0.f;
  const ScoreCtx sc = score_ctx(a);
#pragma unroll
  for (int c = 0; c < NC; ++c) live_frag(fq[c], c, h, a.dh, w.live);
  settle(w.slope), settle(w.doc);
  while (t < tiles) {
    const int k0 = t * BK, tn = t + workers;
    const int doc = kdoc && lane < BK && k0 + lane < a.Lk ? kdoc[k0 + lane] : -1;
    const Place at = place(a, k0 - wb.p_max, k0 + BK - 1 - wb.p_min);
    // requests complete in order: all but the newest tile (the values asked for after these keys, the keys asked for after these values)
    dma_wait<dv.N>();
    dk.clear_pads(sK, a.dh);
    float x[16];
    fwd_products<T, D, true, 1>(x, fq, sK, lane, a.dh);
    wave_sync();                                          // the keys have been read
    if (tn < tiles) dk.load(lds, tn * BK);
    if (kdoc) {
      if (lane < BK) sDoc[lane] = doc;
      wave_sync();
    }
    fwd_softmax<T, D, MOD, true, 1>(st, x, k0, w, a, sc, tab, bias.bucket, at, k0 + BK > wb.hi_min || kdoc, kdoc ? sDoc : nullptr, h);
    if (tn < tiles) dma_wait<dk.N>();
    else dma_wait<0>();
    if (k0 + BK > len || kdoc) {
      zero_rows<T, D, BK, 64>(sV, len - k0, kdoc ? sDoc : nullptr);
      wave_sync();
    }
    fwd_values<T, D, 1>(st, x, sV, lane);
    wave_sync();                                          // the values have been read
    if (tn < tiles) dv.load(lds + TILE, tn * BK);
    t = tn;
  }
  // join the waves: weights 2^(m_w - max m); accumulators through LDS (the tiles are done with)
  __syncthreads();
  float *sM = (float *)smem, *sL = sM + 64 * WAVES, *sA = sL + 64 * WAVES;       // [wave][lane], [wave][register][lane]
  sM[wave * 64 + lane] = st.m;
  __syncthreads();
  float m = sM[lane];
#pragma unroll
  for (int u = 1; u < WAVES; ++u) m = fmaxf(m, sM[u * 64 + lane]);
  const float f = m == -INFINITY ? 0.f : ex2(st.m - m);
  st.m = m;
  sL[wave * 64 + lane] = st.l * f;
  // one block of 32 dimensions at a time; wave u adds the four waves' copies of block u and keeps the sum
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) sA[((wave * ND + d) * 16 + i) * 64 + lane] = st.acc[d][i] * f;
  __syncthreads();
  st.l = sL[lane] + sL[64 + lane] + sL[128 + lane] + sL[192 + lane];
  if (wave != 0) return;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = 0.f;
#pragma unroll
      for (int u = 0; u < WAVES; ++u) v += sA[((u * ND + d) * 16 + i) * 64 + lane];
      st.acc[d][i] = v;
    }
  fwd_store(g, st, w, b, split, h);
}

// Joins the splits of a row: weights 2^(m_s - max m).  One wave per row: four groups of 16 lanes (8 elements each) take every fourth
// split and are added in a fixed order.  Bound by the latency of a few loads: 7 us for 2048 rows of 128 and 16 splits (17 MB).
template <typename T> __global__ void __launch_bounds__(256) mmt_long_attn_join_kernel(const Args g) {
  const mmt_long_attention &a = g.a;
  const int64_t rows = (int64_t)a.B * a.H * a.Lq, r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int lane = threadIdx.x & 63, sub = lane >> 4, d0 = (lane & 15) * 8;
  float m = -INFINITY;
  for (int s = lane; s < g.nsplit; s += 64) m = fmaxf(m, g.part_ml[2 * (s * rows + r)]);
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
  const float ms = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 o[2] = {};
#pragma unroll 4
  for (int s = sub; s < g.nsplit; s += 4) {
    const int64_t rs = s * rows + r;
    const float ls = g.part_ml[2 * rs + 1], f = ls == 0.f ? 0.f : ex2(g.part_ml[2 * rs] - ms);
    f32x4 p[2] = {};
    if (d0 < a.dh) p[0] = *(const f32x4 *)(g.part_o + rs * a.dh + d0), p[1] = *(const f32x4 *)(g.part_o + rs * a.dh + d0 + 4);
    l = fmaf(ls, f, l);
    if (ls != 0.f) o[0] += p[0] * f, o[1] += p[1] * f;   // (a split without keys may hold anything)
  }
#pragma unroll
  for (int k = 16; k < 64; k <<= 1) {
    l += __shfl_xor(l, k);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e >> 2][e & 3] += __shfl_xor(o[e >> 2][e & 3], k);
  }
  const bool some = l != 0.f;
  const float inv = some ? 1.f / l : 0.f;
  const int64_t i = r % a.Lq, bh = r / a.Lq, hd = bh % a.H, b = bh / a.H;
  if (g.lse && lane == 0) g.lse[r] = some ? (m + log2f(l * ex2(-Elem<T>::PSHIFT))) * LN2 : -INFINITY;
  if (sub == 0 && d0 < a.dh) {
    typename Elem<T>::V8 v, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = some ? o[e >> 2][e & 3] * inv : 0.f;
      v[e] = (T)y, lo[e] = (T)(y - (float)v[e]);
    }
    const int64_t at = ((b * a.Lq + i) * a.H + hd) * a.dh + d0;
    *(typename Elem<T>::V8 *)((T *)g.out + at) = v;
    if (g.low) *(typename Elem<T>::V8 *)((T *)g.low + at) = lo;
  }
}

// document ids -> per tile of `bk`: smallest, largest live id, and whether any row of the tile is dead or missing.  Entries 0 .. nk - 1
// are of the keys, the rest of the queries.
template <typename T> __global__ void mmt_long_attn_docs_kernel(const Args g, int bk, int nk, int total, DocRange *out) {
  int n = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, at = n;
  if (n >= total) return;
  const bool key = n < nk;
  if (!key) n -= nk;
  const int L = key ? g.a.Lk : g.a.Lq, nt = (L + bk - 1) / bk, t = n % nt, j = t * bk + lane;
  const int *doc = key ? g.a.k_doc : g.a.q_doc;
  const int id = lane < bk && j < L ? doc[(int64_t)(n / nt) * L + j] : -1;
  const int lo = wave_min(id >= 0 ? id : 0x7fffffff), hi = wave_max(id);
  const bool dead = __any(lane < bk && id < 0);
  if (lane == 0) out[at] = DocRange{lo, hi, dead ? 1 : 0, 0};
}

// --------------------------------------------------------------------------------------------------------------- backward
//   dV = P^T dO;   dP = dO V^T;   dU = P (dP - delta), delta_i = rowsum(dO o) - dlse_i;   dS = dU (1 - tanh^2)
//   dQ = scale dS K;   dK = scale dS^T Q;   dtable[h][b] = sum of dU over the pairs of the bucket
// Two kernels recompute the probabilities from the saved log-sum: one walks the keys of a query tile (dQ), the other the queries of
// a key tile (dK, dV, summed over the query heads that share the key head).  Seven products instead of the five of a single pass,
// but every sum has a fixed order and an owner: no atomics, the same bits every time.
// delta decides the sign and size of dU where a row sees few keys.  It starts from out and what rounding took from it (`low`, which the
// forward keeps for this); P itself was rounded on its way into out, but the sum of dU over a row has to be dlse: what it is instead is
// the error of delta, and the dQ kernel corrects it for everything that comes after.

// fp16: the score gradients are rounded to 5 exponent bits, so they are first multiplied by a power of two that takes their bound
// 2 max|do_i| max|v_j| + max|dlse| to at most 2^15; each workgroup leaves its part of the three maxima.  16 lanes per row.
template <typename T> __global__ void __launch_bounds__(STAT_THREADS) mmt_long_attn_maxima_kernel(const Args g, f32x4 *maxima) {
  const mmt_long_attention &a = g.a;
  typedef typename Elem<T>::V8 V8;
  const int64_t rows = (int64_t)a.B * a.H * a.Lq, vrows = (int64_t)a.B * a.Lk * a.Hk;
  const int d0 = (threadIdx.x & 15) * 8;
  float m[3] = {0.f, 0.f, 0.f};
  auto square = [&](const T *row) {
    float s = 0.f;
    if (d0 < a.dh) {
      const V8 v = *(const V8 *)(row + d0);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf((float)v[e], (float)v[e], s);
    }
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) s += __shfl_xor(s, k);
    return isfinite(s) ? s : 0.f;
  };
  for (int64_t r = (int64_t)blockIdx.x * STAT_ROWS + (threadIdx.x >> 4); r < rows; r += (int64_t)gridDim.x * STAT_ROWS) {
    const int64_t hd = r % a.H, bi = r / a.H, i = bi % a.Lq, b = bi / a.Lq;
    if (a.q_doc && a.q_doc[b * a.Lq + i] < 0) continue;
    const float dl = g.dlse ? fabsf(g.dlse[(b * a.H + hd) * a.Lq + i]) : 0.f, lse = g.lse[(b * a.H + hd) * a.Lq + i];
    const float norm = square((const T *)g.dout + b * g.do_bs + i * g.do_rs + hd * g.do_hs);
    if (lse == -INFINITY) continue;                       // (sees nothing: takes no part)
    m[0] = fmaxf(m[0], norm);
    if (isfinite(dl)) m[2] = fmaxf(m[2], dl);
  }
  for (int64_t r = (int64_t)blockIdx.x * STAT_ROWS + (threadIdx.x >> 4); r < vrows; r += (int64_t)gridDim.x * STAT_ROWS) {
    const int64_t hd = r % a.Hk, bj = r / a.Hk, j = bj % a.Lk, b = bj / a.Lk;
    if (j >= row_len(a, (int)b) || (a.k_doc && a.k_doc[b * a.Lk + j] < 0)) continue;
    m[1] = fmaxf(m[1], square((const T *)a.v + b * a.v_bs + j * a.v_rs + hd * a.v_hs));
  }
#pragma unroll
  for (int k = 16; k < 64; k <<= 1)
    for (int e = 0; e < 3; ++e) m[e] = fmaxf(m[e], __shfl_xor(m[e], k));
  __shared__ f32x4 part[STAT_THREADS / 64];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = f32x4{m[0], m[1], m[2], 0.f};
  __syncthreads();
  if (threadIdx.x == 0) {
    f32x4 v = part[0];
    for (int w = 1; w < STAT_THREADS / 64; ++w)
      for (int e = 0; e < 3; ++e) v[e] = fmaxf(v[e], part[w][e]);
    maxima[blockIdx.x] = v;
  }
}
// each wave of the dQ kernel reads them all (4 KiB; a kernel in between cost 6 us and a launch)
__device__ __forceinline__ float score_grad_scale(const f32x4 *maxima, int parts) {
  f32x4 v = {};
#pragma unroll
  for (int n = 0; n < STAT_PARTS / 64; ++n) {
    const f32x4 u = maxima[min(n * 64 + (int)(threadIdx.x & 63), parts - 1)];
    for (int e = 0; e < 3; ++e) v[e] = fmaxf(v[e], u[e]);
  }
  for (int m = 1; m < 64; m <<= 1)
    for (int e = 0; e < 3; ++e) v[e] = fmaxf(v[e], __shfl_xor(v[e], m));
  const float bound = 2.f * sqrtf(v[0]) * sqrtf(v[1]) + v[2];
  int e = 0;
  const bool known = bound > 0.f && isfinite(bound);
  if (known) (void)frexpf(bound, &e);                                     // bound < 2^e
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(ldexpf(1.f, known ? max(-60, min(60, 15 - e)) : 0))));
}

// dQ, and the statistics of the rows for the other kernels: log-sum in units of log 2 (+inf for a row without keys: its probabilities
// are 0) and the corrected delta.  The forward's geometry; K is read twice from LDS (as rows for the scores, transposed for
// dQ^T += K^T dS^T), V once. Where a workgroup's rows see at most TWICE tiles (the beginnings of causal rows and of documents, short
// rows), 16-bit types go over them twice, the first time for delta alone: a probability's rounding does not average out over few keys.
// Packed scenes of 300 to 800 tokens (2 x 4096, 16 heads of 64): dQ is 0.0025 off with one pass for all, in 65 us, 0.0024 with two up to 8
// tiles, in 82, and with two for all, in 112; 0.0023 is what the roundings of dS and of dQ itself make.  fp32 rounds no probability.
// Bound like the forward: 472 us for its causal case of 8192 tokens (870 TFLOP/s), 81 us for the one of 2048.
// With a learned bias the kernel also sums dU over the tiles that lie wholly beyond the reach on either side.
constexpr int TWICE = 8;
template <typename T, int D, bool GAPS, bool MOD, int TEAMS>
__global__ void __launch_bounds__(TEAMS * THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_dq_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BK = L::BK, NK = BK / 32, NC = D / 16, ND = D / 32, AT_ONCE = D > 64 ? 1 : NK;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  int *sDoc2 = (int *)(smem + TEAMS * 4 * L::BYTES), *sB = sDoc2 + TEAMS * 2 * BK;
  const Lut lut = {(float *)(sB + 6 * WAVES) + a.reach + PAD};
  const int grp = blockIdx.x % g.groups, n = blockIdx.x / g.groups, gi = n % g.G;
  int qt = n / g.G;
  if (a.causal) qt = g.nqt - 1 - qt;
  const int kh = grp % a.Hk, b = grp / a.Hk, head = kh * g.G + gi;
  const int lane = threadIdx.x & 63, w_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = w_all % WAVES, team = w_all / WAVES, h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b), prefix = a.prefix ? scalar_load(a.prefix + b) : 0;
  Row w = make_row(g, b, head, qt * ROWS + wave * 32 + col, len, prefix);
  const int64_t r = ((int64_t)b * a.H + head) * a.Lq + min(w.i, a.Lq - 1);
  const T *qrow = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)min(w.i, a.Lq - 1) * a.q_rs + (int64_t)head * a.q_hs;
  const T *drow = (const T *)g.dout + (int64_t)b * g.do_bs + (int64_t)min(w.i, a.Lq - 1) * g.do_rs + (int64_t)head * g.do_hs;
  const int64_t orow = (((int64_t)b * a.Lq + min(w.i, a.Lq - 1)) * a.H + head) * a.dh;
  V8 fq[NC], fd[NC];
  float delta = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    fq[c] = mem_frag<T>(qrow, c, h, a.dh);
    fd[c] = mem_frag<T>(drow, c, h, a.dh);
  }
  float dl = g.dlse ? g.dlse[r] : 0.f, lse = g.lse[r];
  const DocRange *rng = g.krng ? g.krng + (int64_t)b * g.nkt : nullptr;
  const int *kdoc = a.k_doc ? a.k_doc + (int64_t)b * a.Lk : nullptr;
  const DocRange ranges = TileIter::ahead(rng, 0, g.nkt);
  Bounds wb, gb;
  if (rng) wb = wave_bounds(w), gb = group_bounds(wb, sB, wave);
  else wb = range_bounds(g, qt * ROWS + wave * 32, 32, len, prefix), gb = range_bounds(g, qt * ROWS, ROWS, len, prefix);
  const int tiles = (gb.hi_max + BK - 1) / BK;
  char *const tiles_at = smem + team * 4 * L::BYTES;
  const unsigned lds = lds_address(tiles_at);
  Dma<T, D> dk, dv;
  dk.init((const T *)a.k + (int64_t)b * a.k_bs + (int64_t)kh * a.k_hs, a.k_rs, a.Lk, a.dh);
  dv.init((const T *)a.v + (int64_t)b * a.v_bs + (int64_t)kh * a.v_hs, a.v_rs, a.Lk, a.dh);
  Deal<TEAMS> deal;
  int ids = 0;                                           // ids: the document of the tile's key `lane`
  auto first = [&](DocRange ready) {
    deal.it.start(rng, gb.d_min, gb.d_max, 0, tiles, ready);
    deal.next(team, BK, len);
    if (deal.t >= 0) {
      dk.load(lds, deal.t * BK);
      dv.load(lds + L::BYTES, deal.t * BK);
      if (kdoc) ids = kdoc[min(deal.t * BK + lane, a.Lk - 1)];
    }
  };
  first(ranges);
  if (MOD && a.rel_bias) lut.fill<TEAMS * THREADS>(a, head);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    V8 o = mem_frag<T>((const T *)g.out + orow, c, h, a.dh), lo = {};
    if (g.low) lo = mem_frag<T>((const T *)g.low + orow, c, h, a.dh);
    live_frag(fq[c], c, h, a.dh, w.live), live_frag(fd[c], c, h, a.dh, w.live);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta = fmaf((float)o[e] + (float)lo[e], (float)fd[c][e], delta);
  }
  // A row that sees nothing takes no part, whatever arrives as its gradient (a squared log-sum's is -inf)
  w.live = w.live && lse != -INFINITY;
  dl = w.live ? dl : 0.f;
  delta = w.live ? half_sum(delta) - dl : 0.f;
  lse = w.live ? lse * LOG2E : INFINITY;
  settle(lse), settle(w.slope), settle(w.doc);
  deal.it.here();
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  const ScoreCtx sc = score_ctx(a);
  float dscale = 1.f;
  if constexpr (Elem<T>::PSHIFT != 0.f) {
    dscale = score_grad_scale(g.maxima, g.stat_parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *g.dscale = dscale;
  }
  float all_u = 0.f, all_p = 0.f, far_u[2] = {0.f, 0.f}, far_p[2] = {0.f, 0.f};

  const bool twice = sizeof(T) == 2 && deal.lead >= 0 && deal.it.at_most(TWICE - TEAMS);
  for (int pass = twice ? 0 : 1; pass < 2; ++pass) {
    auto step = [&](auto buffer) {
      constexpr int buf = decltype(buffer)::value;
      const int k0 = deal.t * BK;
      const bool mine = TEAMS == 1 || deal.t >= 0, mixed = deal.mixed, zero = deal.zero, any_zero = deal.any_zero;
      char *sK = tiles_at + buf * 2 * L::BYTES, *sV = sK + L::BYTES;
      int *sDoc = sDoc2 + (TEAMS == 1 ? buf : team * 2 + buf) * BK;
      if (kdoc && wave == 0 && lane < BK) sDoc[lane] = ids;
      dma_wait<0>();
      if constexpr (GAPS) dk.clear_pads(sK, a.dh), dv.clear_pads(sV, a.dh);
      __syncthreads();
      if (any_zero) {
        if (zero) {
          zero_rows<T, D>(sK, len - k0, mixed ? sDoc : nullptr);
          zero_rows<T, D>(sV, len - k0, mixed ? sDoc : nullptr);
        }
        __syncthreads();
      }
      deal.next(team, BK, len);
      if (deal.t >= 0) {
        dk.load(lds + (buf ^ 1) * 2 * L::BYTES, deal.t * BK);
        dv.load(lds + (buf ^ 1) * 2 * L::BYTES + L::BYTES, deal.t * BK);
        if (kdoc) ids = kdoc[min(deal.t * BK + lane, a.Lk - 1)];
      }
      if (mine && k0 < wb.hi_max) {
        const bool need_mask = k0 + BK > wb.hi_min || mixed;
        // by the whole workgroup's rows: the table kernel takes the tiles that are left with the same rule
        const Place at = place(a, k0 - gb.p_max, k0 + BK - 1 - gb.p_min);
#pragma unroll AT_ONCE
        for (int kt = 0; kt < NK; ++kt) {
          // (the two products one after the other where registers are short: what is live grows with how far the compiler pulls them together)
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (has_chunk<GAPS, NC>(c, a.dh)) s = Elem<T>::mma(row_frag<T, D>(sK, 32 * kt + col, c, h), fq[c], s);
          float x[16], th[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = s[i];
          Linear f = {sc.c_scale, 0.f};
          if constexpr (MOD) f = modify<1, true, false>(a, sc, x, th, k0 + 32 * kt + 4 * h - w.p, w.slope, lut.mid, nullptr, at);
          if (need_mask) mask_keys(x, k0 + 32 * kt, w.hi, mixed ? sDoc + 32 * kt : nullptr, w.doc, h);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = ex2(fmaf(x[i], f.mul, f.add - lse));
          if constexpr (D > 64) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (has_chunk<GAPS, NC>(c, a.dh)) dp = Elem<T>::mma(row_frag<T, D>(sV, 32 * kt + col, c, h), fd[c], dp);
          float su = 0.f, sp = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (MOD) sp += x[i];
            x[i] *= dp[i] - delta;
            su += x[i];
          }
          all_u += su;
          if (pass == 0) continue;
          if (MOD) all_p += sp;
          if (MOD && a.rel_bias) {
            if (at.far < 0) far_u[0] += su, far_p[0] += sp;
            if (at.far > 0) far_u[1] += su, far_p[1] += sp;
          }
          if (MOD && sc.capped) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= fmaf(-th[i], th[i], 1.f);
          }
          if constexpr (Elem<T>::PSHIFT != 0.f) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= dscale;
          }
          if constexpr (D > 64) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const V8 ds = round8<T>(x + 8 * c);
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] = Elem<T>::mma(col_frag<T, D>(sK, 32 * kt + 16 * c, d, lane), ds, acc[d]);
          }
        }
      }
        };
    while (deal.lead >= 0) {
      step(Const<0>());
      if (deal.lead < 0) break;
      step(Const<1>());
    }
    // the sum of dU over a row is dlse (0 without it) by definition: what it is instead is the error of delta
    all_u = half_sum(all_u);
    if constexpr (TEAMS == 2) {
      float *s = (float *)smem;
      __syncthreads();                                      // (the tiles are done with)
      s[threadIdx.x] = all_u;
      __syncthreads();
      all_u = s[threadIdx.x % THREADS] + s[THREADS + threadIdx.x % THREADS];
    }
    all_u = lse == INFINITY ? 0.f : all_u - dl;
    if (pass == 0) {
      delta += all_u;
      all_u = 0.f;
      __syncthreads();                                      // (the buffers are filled anew)
      first(TileIter::ahead(rng, 0, g.nkt));
    }
  }
  if (MOD && a.rel_bias) {                                  // what the probabilities sum to, instead of 1: lse is rounded at its own size
    all_p = half_sum(all_p);
    if constexpr (TEAMS == 2) {
      float *s = (float *)smem + 2 * THREADS;
      s[threadIdx.x] = all_p;
      __syncthreads();
      all_p = s[threadIdx.x % THREADS] + s[THREADS + threadIdx.x % THREADS];
    }
    all_p = all_p > 0.f ? 1.f / all_p : 1.f;
    if (w.valid && h == 0 && team == 0) g.norm[r] = all_p;
  }
  if (w.valid && h == 0 && team == 0) g.stat[r] = make_float2(lse, delta + all_u);
  if (MOD && a.rel_bias) {
#pragma unroll
    for (int s = 0; s < 2; ++s) far_u[s] = wave_sum(w.live ? (far_u[s] - all_u * far_p[s]) * all_p : 0.f);
    __syncthreads();
    float *sF = (float *)sB;
    if (lane == 0) sF[2 * w_all] = far_u[0], sF[2 * w_all + 1] = far_u[1];
    __syncthreads();
    if (threadIdx.x < 2) {
      float v = 0.f;
      for (int u = 0; u < TEAMS * WAVES; ++u) v += sF[2 * u + threadIdx.x];
      // item order (b, qt, head) for the reduction, whatever order the workgroups ran in
      g.far_part[(((int64_t)b * g.nqt + qt) * a.H + head) * 2 + threadIdx.x] = v;
    }
  }
  if constexpr (TEAMS == 2) {
    float *s = (float *)smem + threadIdx.x % THREADS;
    __syncthreads();
    if (team) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[(16 * d + i) * THREADS] = acc[d][i];
    }
    __syncthreads();
    if (team) return;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] += s[(16 * d + i) * THREADS];
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

// dK, dV.  A wave owns 32 keys (the accumulator's columns; their rows of K and V stay in registers as operands), the queries of the
// heads that share the key head go by in LDS tiles, as rows for S and dP and transposed for dV^T += dO^T P and dK^T += Q^T dS.
// With few key tiles the query heads and the queries are dealt over zh x zq parts, which a second kernel adds up in order.
// For fp32, and 16-bit types up to a head size of 64: K, V, dK and dV of 32 keys take 192 registers at 128, which leaves room for one wave
// per SIMD (8192 causal tokens x 16 heads: 1380 us with one, 2470 with two and spills, the next kernel's 618).  Up to 64 this one is: bf16
// 2 x 2048 x 16 heads of 64 93 us, the next one 118; 2 x 4096 tokens in packed scenes 79, the next one 91.  Bound by vector instructions
// and the latency between them, at two waves per SIMD: 740 TFLOP/s in the first case.
template <typename T, int D, bool GAPS, bool MOD>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_dkv_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BQ = L::BK, NQ = BQ / 32, NC = D / 16, ND = D / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  float *sStat2 = (float *)(smem + 4 * L::BYTES);         // [2][log-sum, delta][BQ]
  int *sDoc2 = (int *)(sStat2 + 4 * BQ), *sB = sDoc2 + 2 * BQ, *sPart = sB + 2 * WAVES;      // sPart: [2], not all rows of the tile take part
  const Lut lut = {(float *)(sB + 6 * WAVES) + a.reach + PAD};
  const int grp = blockIdx.x % g.groups;
  int n = blockIdx.x / g.groups;
  const int z = n % (g.zh * g.zq), zh = z % g.zh, zq = z / g.zh;
  const int kt = n / (g.zh * g.zq);                       // causal: the first keys are seen by the most queries
  const int kh = grp % a.Hk, b = grp / a.Hk, head0 = kh * g.G;
  const int g_per = (g.G + g.zh - 1) / g.zh, g0 = zh * g_per, g1 = min(g.G, g0 + g_per);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b), off = len - a.Lq, prefix = a.prefix ? scalar_load(a.prefix + b) : 0;
  const int j = kt * ROWS + wave * 32 + col;
  const int kdoc = a.k_doc ? a.k_doc[(int64_t)b * a.Lk + min(j, a.Lk - 1)] : 0;
  const T *krow = (const T *)a.k + (int64_t)b * a.k_bs + (int64_t)min(j, a.Lk - 1) * a.k_rs + (int64_t)kh * a.k_hs;
  const T *vrow = (const T *)a.v + (int64_t)b * a.v_bs + (int64_t)min(j, a.Lk - 1) * a.v_rs + (int64_t)kh * a.v_hs;
  V8 fk[NC], fv[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    fk[c] = mem_frag<T>(krow, c, h, a.dh);
    fv[c] = mem_frag<T>(vrow, c, h, a.dh);
  }
  // queries that may see a key of this workgroup: position >= its first key, unless the prefix reaches into it
  const int i_first = a.causal && prefix <= kt * ROWS ? max(0, kt * ROWS - off) : 0;
  const int all0 = min(i_first, a.Lq) / BQ, all1 = kt * ROWS < len ? (a.Lq + BQ - 1) / BQ : 0;
  const int t_per = (max(0, all1 - all0) + g.zq - 1) / g.zq, t0 = all0 + zq * t_per, t1 = min(all1, t0 + t_per);
  const int n_qt = (a.Lq + BQ - 1) / BQ;
  const DocRange *rng = g.qrng ? g.qrng + (int64_t)b * n_qt : nullptr;
  const DocRange ranges = TileIter::ahead(rng, t0, n_qt);
  const bool live = j < len && kdoc >= 0;
  const int j_lo = kt * ROWS + wave * 32;                 // first key of the wave
  const bool all_live = __all(live);
  int gd_min = 0, gd_max = 0;
  if (rng) {
    const int d_min = wave_min(live ? kdoc : 0x7fffffff), d_max = wave_max(live ? kdoc : -1);
    if (lane == 0) sB[2 * wave] = d_min, sB[2 * wave + 1] = d_max;
    __syncthreads();
    gd_min = 0x7fffffff, gd_max = -1;
    for (int v = 0; v < WAVES; ++v) gd_min = min(gd_min, sB[2 * v]), gd_max = max(gd_max, sB[2 * v + 1]);
    gd_min = __builtin_amdgcn_readfirstlane(gd_min), gd_max = __builtin_amdgcn_readfirstlane(gd_max);
  }

  f32x16 acck[ND], accv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acck[d] = f32x16{}, accv[d] = f32x16{};
  const ScoreCtx sc = score_ctx(a);
  // fp16: P is rounded times 2^PSHIFT; the surplus is taken out of dS again together with its own scaling
  const float dscale = Elem<T>::PSHIFT != 0.f ? scalar_load(g.dscale) : 1.f;
  const float ds_mul = dscale * ex2(-Elem<T>::PSHIFT);

  const int *qdoc = a.q_doc ? a.q_doc + (int64_t)b * a.Lq : nullptr;
  const unsigned lds = lds_address(smem);
  Dma<T, D> dmq, dmo;
  dmq.init((const T *)a.q + (int64_t)b * a.q_bs + (int64_t)head0 * a.q_hs, a.q_rs, a.Lq, a.dh);
  dmo.init((const T *)g.dout + (int64_t)b * g.do_bs + (int64_t)head0 * g.do_hs, g.do_rs, a.Lq, a.dh);
  const char *qbase = dmq.base, *obase = dmo.base;

  // the tiles of all heads as one sequence, so that the next head's first tile is on its way during this head's last
  TileIter it;
  int gi = g0 - 1, t = -1, lut_gi = -1;
  const float2 *stat = nullptr;
  float2 st_next = make_float2(INFINITY, 0.f);
  float slope_next = 0.f;
  int doc_next = -1;
  auto advance = [&](auto at_start) {                                  // next tile, over head ends; -1 at the end
    int n = gi < g0 ? -1 : it.next();
    while (n < 0 && ++gi < g1) {
      stat = g.stat + ((int64_t)b * a.H + head0 + gi) * a.Lq;
      dmq.base = qbase + (int64_t)gi * a.q_hs * (int64_t)sizeof(T);
      dmo.base = obase + (int64_t)gi * g.do_hs * (int64_t)sizeof(T);
      if (MOD && a.slopes) slope_next = scalar_load(a.slopes + head0 + gi) * LOG2E;
      it.start(rng, gd_min, gd_max, t0, t1, decltype(at_start)::value && gi == g0 ? ranges : TileIter::ahead(rng, t0, n_qt));
      n = it.next();
    }
    return n;
  };
  auto fetch = [&](int tile, int to) {
    dmq.load(lds + to * 2 * L::BYTES, tile * BQ);
    dmo.load(lds + to * 2 * L::BYTES + L::BYTES, tile * BQ);
    if (threadIdx.x < BQ) {
      // (neither waits for the other, or for the tile: rows that are missing or dead are sorted out when the tile is here)
      const int i = min(tile * BQ + (int)threadIdx.x, a.Lq - 1);
      doc_next = qdoc ? qdoc[i] : 0;
      st_next = stat[i];
    }
  };
  t = advance(Const<1>());
  if (t >= 0) fetch(t, 0);
#pragma unroll
  for (int c = 0; c < NC; ++c) live_frag(fk[c], c, h, a.dh, live), live_frag(fv[c], c, h, a.dh, live);
  it.here();
  auto step = [&](auto buffer) {
    constexpr int buf = decltype(buffer)::value;
    const int q0 = t * BQ, head = head0 + gi;
    char *sQ = smem + buf * 2 * L::BYTES, *sO = sQ + L::BYTES;
    float *sStat = sStat2 + buf * 2 * BQ;
    int *sDoc = sDoc2 + buf * BQ;
    const bool docs = it.mixed();
    const int cur_gi = gi;
    const float slope = slope_next;
    if (threadIdx.x < BQ) {
      const int doc = q0 + (int)threadIdx.x < a.Lq && st_next.x != INFINITY ? doc_next : -1;      // negative: takes no part
      sDoc[threadIdx.x] = doc;
      sStat[threadIdx.x] = doc >= 0 ? st_next.x : INFINITY, sStat[BQ + threadIdx.x] = doc >= 0 ? st_next.y : 0.f;
      const bool out = __any(doc < 0);
      if (threadIdx.x == 0) sPart[buf] = out;
    }
    dma_wait<0>();
    if constexpr (GAPS) dmq.clear_pads(sQ, a.dh), dmo.clear_pads(sO, a.dh);
    __syncthreads();
    if (MOD && a.rel_bias && lut_gi != cur_gi) {          // another head's bias
      lut.fill(a, head);
      lut_gi = cur_gi;
      __syncthreads();
    }
    // rows that take no part - missing, padding, or seeing nothing - are cleared (0 x inf would reach all keys) and masked (a cleared
    // row's product with an infinite key is NaN)
    const bool part = __builtin_amdgcn_readfirstlane(sPart[buf]) != 0, mixed = docs || part;
    if (part) {
      zero_rows<T, D>(sQ, BQ, sDoc);
      zero_rows<T, D>(sO, BQ, sDoc);
      __syncthreads();
    }
    const int tn = advance(Const<0>());
    if (tn >= 0) fetch(tn, buf ^ 1);
    const int p0 = off + q0;
    // the last row of the tile sees the most
    if (!a.causal || max(p0 + BQ, prefix) > j_lo) {
      const bool need_mask = mixed || !all_live || (a.causal && max(p0 + 1, prefix) < j_lo + 32);
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (!has_chunk<GAPS, NC>(c, a.dh)) continue;
          s = Elem<T>::mma(row_frag<T, D>(sQ, 32 * qt + col, c, h), fk[c], s);
          dp = Elem<T>::mma(row_frag<T, D>(sO, 32 * qt + col, c, h), fv[c], dp);
        }
        float x[16], th[16], p[16];
        Linear f = {sc.c_scale, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = s[i];
        if constexpr (MOD) {
          const int pq = p0 + 32 * qt;
          f = modify<-1, true, false>(a, sc, x, th, j - pq - 4 * h, slope, lut.mid, nullptr, place(a, j_lo - pq - 31, j_lo + 31 - pq));
        }
        f.add += Elem<T>::PSHIFT;
        f32x4 st[4];
        acc_rows(st, sStat + 32 * qt, h);
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = ex2(fmaf(x[i], f.mul, f.add - st[i >> 2][i & 3]));
        if (need_mask) {
          const int lo = a.causal ? (j < prefix ? 0 : j - off - q0 - 32 * qt) : -(1 << 30);      // first row of the sub-tile that sees key j
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = (live & (acc_row(i, h) >= lo)) ? p[i] : 0.f;
          if (mixed) {
            int id[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) id[i] = sDoc[32 * qt + acc_row(i, h)];
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = id[i] == kdoc ? p[i] : 0.f;
          }
        }
        acc_rows(st, sStat + BQ + 32 * qt, h);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = p[i] * (dp[i] - st[i >> 2][i & 3]);
        if (MOD && sc.capped) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= fmaf(-th[i], th[i], 1.f);
        }
        if constexpr (Elem<T>::PSHIFT != 0.f) {
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
    }
    t = tn;
  };
  while (t >= 0) {
    step(Const<0>());
    if (t < 0) break;
    step(Const<1>());
  }
  if (j >= a.Lk) return;
  const int64_t o = (((int64_t)b * a.Lk + j) * a.Hk + kh) * a.dh, part = (int64_t)a.B * a.Lk * a.Hk * a.dh * z;
  const float f_k = a.scale / dscale, f_v = ex2(-Elem<T>::PSHIFT);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int dim = 32 * d + 8 * q + 4 * h;
      if (dim >= a.dh) continue;
      f32x4 vk, vv;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        vk[e] = live ? acck[d][4 * q + e] * f_k : 0.f;
        vv[e] = live ? accv[d][4 * q + e] * f_v : 0.f;
      }
      if (g.part_dk) {
        *(f32x4 *)(g.part_dk + part + o + dim) = vk;
        *(f32x4 *)(g.part_dv + part + o + dim) = vv;
      } else {
        *(typename Elem<T>::V4 *)((T *)g.dk + o + dim) = __builtin_convertvector(vk, typename Elem<T>::V4);
        *(typename Elem<T>::V4 *)((T *)g.dv + o + dim) = __builtin_convertvector(vv, typename Elem<T>::V4);
      }
    }
}

// dK, dV at head sizes above 64 in 16-bit types.  Keys, their gradients and the products of 32 keys do not fit into the 256 registers
// that two waves per SIMD leave each; so the eight waves of a workgroup (128 keys) share the work in two steps per tile of 64 queries:
//   1. wave w computes P and dS of 32 queries x 32 keys (its K and V rows stay in registers) and leaves them in LDS in the order of
//      the accumulator, which is the order of the second step's operand: 16 bytes per lane, no rearrangement;
//   2. wave w adds up one of the two outputs for KB x 32 keys and a part of the dimensions, with dO or Q read transposed.
// 8192 causal tokens x 16 heads of 128 over 4: 618 us, 890 TFLOP/s for the four products.  About 290 KiB go through LDS per tile, half of
// the time of its matrix instructions (LDS 41 % of the cycles, matrix 37 %, vector 30 %); bound by the steps' order: two barriers per
// tile, one workgroup per CU, and its waves wait for 47 % of the time.  With modified scores at 128, 20 bytes per lane live in scratch (all 256
// registers are taken).
template <typename T, int D, bool GAPS, bool MOD>
__global__ void __launch_bounds__(512, 2) mmt_long_attn_dkv2_kernel(const Args g) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BQ = 64, NC = D / 16, ND = D / 32, KB = ND % 2 ? 1 : 2, NT = ND / KB;      // KB key blocks and NT dimension tiles per wave
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  char *sP = smem + 4 * L::BYTES, *sS = sP + 128 * BQ * 2;                 // [key block][16 queries][lane] x 16 bytes
  float *sStat2 = (float *)(sS + 128 * BQ * 2);                             // [2][log-sum, delta][BQ]
  int *sDoc2 = (int *)(sStat2 + 4 * BQ), *sB = sDoc2 + 2 * BQ, *sPart = sB + 16;      // sPart: [2], not all rows of the tile take part
  const Lut lut = {(float *)(sB + 20) + a.reach + PAD};
  const int grp = blockIdx.x % g.groups;
  int n = blockIdx.x / g.groups;
  const int z = n % (g.zh * g.zq), zh = z % g.zh, zq = z / g.zh;
  const int kt = n / (g.zh * g.zq);                       // causal: the first keys are seen by the most queries
  const int kh = grp % a.Hk, b = grp / a.Hk, head0 = kh * g.G;
  const int g_per = (g.G + g.zh - 1) / g.zh, g0 = zh * g_per, g1 = min(g.G, g0 + g_per);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b), off = len - a.Lq, prefix = a.prefix ? scalar_load(a.prefix + b) : 0;
  const int qh = wave & 1, kb = wave >> 1;                // first step: half of the queries, block of 32 keys
  const int j_lo = kt * ROWS + kb * 32, j = j_lo + col;
  const int kdoc = a.k_doc ? a.k_doc[(int64_t)b * a.Lk + min(j, a.Lk - 1)] : 0;
  const T *krow = (const T *)a.k + (int64_t)b * a.k_bs + (int64_t)min(j, a.Lk - 1) * a.k_rs + (int64_t)kh * a.k_hs;
  const T *vrow = (const T *)a.v + (int64_t)b * a.v_bs + (int64_t)min(j, a.Lk - 1) * a.v_rs + (int64_t)kh * a.v_hs;
  V8 fk[NC], fv[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    fk[c] = mem_frag<T>(krow, c, h, a.dh);
    fv[c] = mem_frag<T>(vrow, c, h, a.dh);
  }
  const int i_first = a.causal && prefix <= kt * ROWS ? max(0, kt * ROWS - off) : 0;
  const int all0 = min(i_first, a.Lq) / BQ, all1 = kt * ROWS < len ? (a.Lq + BQ - 1) / BQ : 0;
  const int t_per = (max(0, all1 - all0) + g.zq - 1) / g.zq, t0 = all0 + zq * t_per, t1 = min(all1, t0 + t_per);
  const int n_qt = (a.Lq + BQ - 1) / BQ;
  const DocRange *rng = g.qrng ? g.qrng + (int64_t)b * n_qt : nullptr;
  const DocRange ranges = TileIter::ahead(rng, t0, n_qt);
  const bool live = j < len && kdoc >= 0;
  const bool all_live = __all(live);
  int gd_min = 0, gd_max = 0;
  if (rng) {
    const int d_min = wave_min(live ? kdoc : 0x7fffffff), d_max = wave_max(live ? kdoc : -1);
    if (lane == 0) sB[2 * wave] = d_min, sB[2 * wave + 1] = d_max;
    __syncthreads();
    gd_min = 0x7fffffff, gd_max = -1;
    for (int v = 0; v < 8; ++v) gd_min = min(gd_min, sB[2 * v]), gd_max = max(gd_max, sB[2 * v + 1]);
    gd_min = __builtin_amdgcn_readfirstlane(gd_min), gd_max = __builtin_amdgcn_readfirstlane(gd_max);
  }

  // second step: which output, which keys (blocks kb2, kb2 + 1, ..), which dimension tiles (dt2, ..)
  const bool to_k = wave & 1;
  const int part = wave >> 1, kb2 = KB == 2 ? 2 * (part & 1) : part, dt2 = KB == 2 ? NT * (part >> 1) : 0;
  f32x16 acc[KB][NT];
#pragma unroll
  for (int k = 0; k < KB; ++k)
#pragma unroll
    for (int d = 0; d < NT; ++d) acc[k][d] = f32x16{};
  const ScoreCtx sc = score_ctx(a);
  const float dscale = Elem<T>::PSHIFT != 0.f ? scalar_load(g.dscale) : 1.f;
  const float ds_mul = dscale * ex2(-Elem<T>::PSHIFT);

  const int *qdoc = a.q_doc ? a.q_doc + (int64_t)b * a.Lq : nullptr;
  const unsigned lds = lds_address(smem);
  Dma<T, D, BQ, 512> dmq, dmo;
  dmq.init((const T *)a.q + (int64_t)b * a.q_bs + (int64_t)head0 * a.q_hs, a.q_rs, a.Lq, a.dh);
  dmo.init((const T *)g.dout + (int64_t)b * g.do_bs + (int64_t)head0 * g.do_hs, g.do_rs, a.Lq, a.dh);
  const char *qbase = dmq.base, *obase = dmo.base;

  // the tiles of all heads as one sequence, so that the next head's first tile is on its way during this head's last
  TileIter it;
  int gi = g0 - 1, t = -1, buf = 0, lut_gi = -1;
  const float2 *stat = nullptr;
  float2 st_next = make_float2(INFINITY, 0.f);
  float slope_next = 0.f;
  int doc_next = -1;
  auto advance = [&](auto at_start) {
    int n = gi < g0 ? -1 : it.next();
    while (n < 0 && ++gi < g1) {
      stat = g.stat + ((int64_t)b * a.H + head0 + gi) * a.Lq;
      dmq.base = qbase + (int64_t)gi * a.q_hs * (int64_t)sizeof(T);
      dmo.base = obase + (int64_t)gi * g.do_hs * (int64_t)sizeof(T);
      if (MOD && a.slopes) slope_next = scalar_load(a.slopes + head0 + gi) * LOG2E;
      it.start(rng, gd_min, gd_max, t0, t1, decltype(at_start)::value && gi == g0 ? ranges : TileIter::ahead(rng, t0, n_qt));
      n = it.next();
    }
    return n;
  };
  auto fetch = [&](int tile, int to) {
    dmq.load(lds + to * 2 * L::BYTES, tile * BQ);
    dmo.load(lds + to * 2 * L::BYTES + L::BYTES, tile * BQ);
    if (threadIdx.x < BQ) {
      // (neither waits for the other, or for the tile: rows that are missing or dead are sorted out when the tile is here)
      const int i = min(tile * BQ + (int)threadIdx.x, a.Lq - 1);
      doc_next = qdoc ? qdoc[i] : 0;
      st_next = stat[i];
    }
  };
  t = advance(Const<1>());
  if (t >= 0) fetch(t, 0);
#pragma unroll
  for (int c = 0; c < NC; ++c) live_frag(fk[c], c, h, a.dh, live), live_frag(fv[c], c, h, a.dh, live);
  it.here();
  while (t >= 0) {
    const int q0 = t * BQ, head = head0 + gi, cur_gi = gi;
    char *sQ = smem + buf * 2 * L::BYTES, *sO = sQ + L::BYTES;
    float *sStat = sStat2 + buf * 2 * BQ;
    int *sDoc = sDoc2 + buf * BQ;
    const bool docs = it.mixed();
    const float slope = slope_next;
    if (threadIdx.x < BQ) {
      const int doc = q0 + (int)threadIdx.x < a.Lq && st_next.x != INFINITY ? doc_next : -1;      // negative: takes no part
      sDoc[threadIdx.x] = doc;
      sStat[threadIdx.x] = doc >= 0 ? st_next.x : INFINITY, sStat[BQ + threadIdx.x] = doc >= 0 ? st_next.y : 0.f;
      const bool out = __any(doc < 0);
      if (threadIdx.x == 0) sPart[buf] = out;
    }
    dma_wait<0>();
    if constexpr (GAPS) dmq.clear_pads(sQ, a.dh), dmo.clear_pads(sO, a.dh);
    __syncthreads();                                      // the tile is here; the last one's second step is done everywhere
    if (MOD && a.rel_bias && lut_gi != cur_gi) {          // another head's bias
      lut.fill<512>(a, head);
      lut_gi = cur_gi;
      __syncthreads();
    }
    // rows that take no part - missing, padding, or seeing nothing - are cleared (0 x inf would reach all keys) and masked (a cleared
    // row's product with an infinite key is NaN)
    const bool part = __builtin_amdgcn_readfirstlane(sPart[buf]) != 0, mixed = docs || part;
    if (part) {
      zero_rows<T, D, BQ, 512>(sQ, BQ, sDoc);
      zero_rows<T, D, BQ, 512>(sO, BQ, sDoc);
      __syncthreads();
    }
    const int tn = advance(Const<0>());
    if (tn >= 0) fetch(tn, buf ^ 1);
    {
      const int p0 = off + q0 + 32 * qh;                  // position of the first of this wave's queries
      const bool need_mask = mixed || !all_live || (a.causal && max(p0 + 1, prefix) < j_lo + 32);
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (has_chunk<GAPS, NC>(c, a.dh)) s = Elem<T>::mma(row_frag<T, D>(sQ, 32 * qh + col, c, h), fk[c], s);
      float x[16], th[16], p[16];
      Linear f = {sc.c_scale, 0.f};
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = s[i];
      if constexpr (MOD) {
        f = modify<-1, true, false>(a, sc, x, th, j - p0 - 4 * h, slope, lut.mid, nullptr, place(a, j_lo - p0 - 31, j_lo + 31 - p0));
      }
      f.add += Elem<T>::PSHIFT;
      f32x4 st[4];
      acc_rows(st, sStat + 32 * qh, h);
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = ex2(fmaf(x[i], f.mul, f.add - st[i >> 2][i & 3]));
      if (need_mask) {
        const int lo = a.causal ? (j < prefix ? 0 : j - p0) : -(1 << 30);      // first of the queries that sees key j
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = (live & (acc_row(i, h) >= lo)) ? p[i] : 0.f;
        if (mixed) {
          int id[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) id[i] = sDoc[32 * qh + acc_row(i, h)];
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = id[i] == kdoc ? p[i] : 0.f;
        }
      }
      __builtin_amdgcn_sched_barrier(0);                  // (keeps the registers of the second product out of the first one's reach)
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (has_chunk<GAPS, NC>(c, a.dh)) dp = Elem<T>::mma(row_frag<T, D>(sO, 32 * qh + col, c, h), fv[c], dp);
      acc_rows(st, sStat + BQ + 32 * qh, h);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = p[i] * (dp[i] - st[i >> 2][i & 3]);
      if (MOD && sc.capped) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= fmaf(-th[i], th[i], 1.f);
      }
      if (Elem<T>::PSHIFT != 0.f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= ds_mul;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int at = ((kb * 4 + qh * 2 + c) * 64 + lane) * 16;
        *(V8 *)(sP + at) = round8<T>(p + 8 * c);
        *(V8 *)(sS + at) = round8<T>(x + 8 * c);
      }
    }
    __syncthreads();                                      // P and dS of the tile are complete
    {
      const char *tr = to_k ? sQ : sO, *op = to_k ? sS : sP;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        V8 fb[KB];
#pragma unroll
        for (int k = 0; k < KB; ++k) fb[k] = *(const V8 *)(op + (((kb2 + k) * 4 + c) * 64 + lane) * 16);
#pragma unroll
        for (int d = 0; d < NT; ++d) {
          const V8 fa = col_frag<T, D>(tr, 16 * c, dt2 + d, lane);
#pragma unroll
          for (int k = 0; k < KB; ++k) acc[k][d] = Elem<T>::mma(fa, fb[k], acc[k][d]);
        }
      }
    }
    t = tn;
    buf ^= 1;
  }
  const float f = to_k ? a.scale / dscale : ex2(-Elem<T>::PSHIFT);
  float *part_out = to_k ? g.part_dk : g.part_dv;
  T *out = (T *)(to_k ? g.dk : g.dv);
#pragma unroll
  for (int k = 0; k < KB; ++k) {
    const int jj = kt * ROWS + (kb2 + k) * 32 + col;
    if (jj >= a.Lk) continue;
    const bool ok = jj < len && !(a.k_doc && a.k_doc[(int64_t)b * a.Lk + jj] < 0);
    const int64_t o = (((int64_t)b * a.Lk + jj) * a.Hk + kh) * a.dh, at = (int64_t)a.B * a.Lk * a.Hk * a.dh * z + o;
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int dim = 32 * (dt2 + d) + 8 * q + 4 * h;
        if (dim >= a.dh) continue;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ok ? acc[k][d][4 * q + e] * f : 0.f;
        if (part_out) *(f32x4 *)(part_out + at + dim) = v;
        else *(typename Elem<T>::V4 *)(out + o + dim) = __builtin_convertvector(v, typename Elem<T>::V4);
      }
  }
}

// the parts of dK and dV, in order; bound by memory (4 parts of 2 x 16.8 MB: 23 us, 6.5 TB/s, part of it still cached)
template <typename T> __global__ void __launch_bounds__(256) mmt_long_attn_dkv_sum_kernel(const Args g) {
  const int64_t n = (int64_t)g.a.B * g.a.Lk * g.a.Hk * g.a.dh, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4 k = {}, v = {};
  for (int z = 0; z < g.zh * g.zq; ++z) {
    k += *(const f32x4 *)(g.part_dk + n * z + i);
    v += *(const f32x4 *)(g.part_dv + n * z + i);
  }
  *(typename Elem<T>::V4 *)((T *)g.dk + i) = __builtin_convertvector(k, typename Elem<T>::V4);
  *(typename Elem<T>::V4 *)((T *)g.dv + i) = __builtin_convertvector(v, typename Elem<T>::V4);
}

// The gradient of the learned bias over the tiles within the reach (the dQ kernel has summed the others).  Sums of millions of
// signed terms that have to come out right to fp32 (30 us for 2 x 2048 x 16 heads of 64 and a reach of 128): dU is recomputed with the exact delta of each row, and every lane adds into
// a column of its own of a [bucket][lane] array in LDS, so that the order of the additions is the program's.  Bound by the latency of
// these load - add - store chains (LDS additions that return nothing took four times as long): four elements at a time are loaded
// together, each of the four then adds all those of its bucket, so that equal buckets store equal sums.  The next tile is on its way
// meanwhile.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 1 : 2) mmt_long_attn_table_kernel(const Args g, float *part) {
  typedef Tile<T, D> L;
  typedef typename Elem<T>::V8 V8;
  constexpr int BK = L::BK, NK = BK / 32, NC = D / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const mmt_long_attention &a = g.a;
  char *sK = smem, *sV = smem + L::BYTES;
  int *sDoc = (int *)(smem + 2 * L::BYTES), *sB = sDoc + 2 * BK;
  const Lut lut = {(float *)(sB + 6 * WAVES) + a.reach + PAD};
  unsigned char *bucket = (unsigned char *)((float *)(sB + 6 * WAVES) + Lut::floats(a)) + a.reach + PAD;   // of distance 0
  float *hist = (float *)(sB + 6 * WAVES) + Lut::floats(a) + ((Lut::floats(a) + 15) & ~15) / 4;
  const int grp = blockIdx.x % g.groups, n = blockIdx.x / g.groups, gi = n % g.G, qt = n / g.G;
  const int kh = grp % a.Hk, b = grp / a.Hk, head = kh * g.G + gi;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int len = row_len(a, b), prefix = a.prefix ? scalar_load(a.prefix + b) : 0;
  Row w = make_row(g, b, head, qt * ROWS + wave * 32 + col, len, prefix);
  const int64_t r = ((int64_t)b * a.H + head) * a.Lq + min(w.i, a.Lq - 1);
  float2 rs = g.stat[r];
  float norm = g.norm[r];
  const T *qrow = (const T *)a.q + (int64_t)b * a.q_bs + (int64_t)min(w.i, a.Lq - 1) * a.q_rs + (int64_t)head * a.q_hs;
  const T *drow = (const T *)g.dout + (int64_t)b * g.do_bs + (int64_t)min(w.i, a.Lq - 1) * g.do_rs + (int64_t)head * g.do_hs;
  V8 fq[NC], fd[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    fq[c] = mem_frag<T>(qrow, c, h, a.dh);
    fd[c] = mem_frag<T>(drow, c, h, a.dh);
  }
  Bounds wb, gb;
  if (g.krng) wb = wave_bounds(w), gb = group_bounds(wb, sB, wave);
  else wb = range_bounds(g, qt * ROWS + wave * 32, 32, len, prefix), gb = range_bounds(g, qt * ROWS, ROWS, len, prefix);
  const ScoreCtx sc = score_ctx(a);
  const int tiles = (gb.hi_max + BK - 1) / BK;
  const DocRange *rng = g.krng ? g.krng + (int64_t)b * g.nkt : nullptr;
  const unsigned lds = lds_address(smem);
  Dma<T, D> dk, dv;
  dk.init((const T *)a.k + (int64_t)b * a.k_bs + (int64_t)kh * a.k_hs, a.k_rs, a.Lk, a.dh);
  dv.init((const T *)a.v + (int64_t)b * a.v_bs + (int64_t)kh * a.v_hs, a.v_rs, a.Lk, a.dh);
  const int *kdoc = a.k_doc ? a.k_doc + (int64_t)b * a.Lk : nullptr;
  // tiles with k0 + BK - 1 - p_min > -reach and k0 - p_max < reach
  int t0 = 0, t1 = 0;
  if (gb.hi_max > 0) {
    t0 = max(0, (gb.p_min - a.reach - BK + 1) / BK);
    while (t0 < tiles && t0 * BK + BK - 1 - gb.p_min <= -a.reach) ++t0;
    t1 = min(tiles, max(0, gb.p_max + a.reach + BK) / BK + 1);
    while (t1 > t0 && (t1 - 1) * BK - gb.p_max >= a.reach) --t1;
  }
  auto next = [&](int t) {                                // the first tile from t on with documents of these rows
    while (t < t1 && rng && (rng[t].lo > gb.d_max || rng[t].hi < gb.d_min)) ++t;
    return t;
  };
  auto request = [&](int t, int *ids) {
    dk.load(lds, t * BK);
    dv.load(lds + L::BYTES, t * BK);
    if (kdoc && threadIdx.x < BK) ids[threadIdx.x] = t * BK + (int)threadIdx.x < a.Lk ? kdoc[t * BK + threadIdx.x] : -1;
  };
  int t = next(t0);
  int *ids = sDoc, *ids_next = sDoc + BK;
  if (t < t1) request(t, ids);
  lut.fill(a, head, bucket);
  float *mine = hist + (int64_t)wave * a.n_buckets * 64 + lane;
  for (int k = 0; k < a.n_buckets; ++k) mine[k * 64] = 0.f;
  w.live = w.live && rs.x != INFINITY;                    // (a row that sees nothing)
#pragma unroll
  for (int c = 0; c < NC; ++c) live_frag(fq[c], c, h, a.dh, w.live), live_frag(fd[c], c, h, a.dh, w.live);
  if (!w.live) w.hi = 0;                                  // (every score masked: a cleared row's product with an infinite key is NaN)
  const float lse2 = w.live ? rs.x : INFINITY, delta = w.live ? rs.y : 0.f;
  settle(w.slope), settle(w.doc), settle(norm);
  while (t < t1) {
    const int k0 = t * BK;
    dma_wait<0>();
    dk.clear_pads(sK, a.dh), dv.clear_pads(sV, a.dh);
    __syncthreads();
    if (k0 + BK > len || kdoc) {
      zero_rows<T, D>(sK, len - k0, kdoc ? ids : nullptr);
      zero_rows<T, D>(sV, len - k0, kdoc ? ids : nullptr);
      __syncthreads();
    }
    f32x16 s[NK], dp[NK];
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
      s[kt] = f32x16{}, dp[kt] = f32x16{};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (!has_chunk<true, NC>(c, a.dh)) continue;
        s[kt] = Elem<T>::mma(row_frag<T, D>(sK, 32 * kt + col, c, h), fq[c], s[kt]);
        dp[kt] = Elem<T>::mma(row_frag<T, D>(sV, 32 * kt + col, c, h), fd[c], dp[kt]);
      }
    }
    __syncthreads();                                      // the products have been taken from the tile
    t = next(t + 1);
    if (t < t1) request(t, ids_next);
    if (k0 < wb.hi_max) {
      const Place at = place(a, k0 - gb.p_max, k0 + BK - 1 - gb.p_min);
#pragma unroll
      for (int kt = 0; kt < NK; ++kt) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = s[kt][i];
        modify<1, false, false>(a, sc, x, nullptr, k0 + 32 * kt + 4 * h - w.p, w.slope, lut.mid, nullptr, at);
        mask_keys(x, k0 + 32 * kt, w.hi, kdoc ? ids + 32 * kt : nullptr, w.doc, h);
        const unsigned char *bk = bucket + max(-a.reach - PAD, min(a.reach + PAD - 27, k0 + 32 * kt + 4 * h - w.p));
        int bucket_of[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) bucket_of[i] = bk[8 * (i >> 2) + (i & 3)];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int *n = bucket_of + 4 * q;
          float u[4], v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = mine[n[e] * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = ex2(x[4 * q + e] - lse2) * norm * (dp[kt][4 * q + e] - delta);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float sum = n[0] == n[e] ? u[0] : 0.f;
#pragma unroll
            for (int f = 1; f < 4; ++f) sum += n[f] == n[e] ? u[f] : 0.f;
            mine[n[e] * 64] = v[e] + sum;
          }
        }
      }
    }
    int *swap = ids;
    ids = ids_next, ids_next = swap;
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
template <typename T> __global__ void mmt_long_attn_table_sum_kernel(const mmt_long_attention a, int64_t n, const float *part, const float *far_part, float *dtable) {
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

// --------------------------------------------------------------------------------------------------------------- launchers
template <typename K> static void launch(K kernel, int64_t grid, size_t lds, hipStream_t st, const Args &g, int threads = THREADS) {
  if (lds > 65536) (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, g);
}

static inline bool modified(const mmt_long_attention &a) { return a.softcap > 0.f || a.slopes || a.rel_bias; }

template <typename T, int D, bool GAPS> static void fwd_size(const Args &g, hipStream_t st) {
  if (g.few) {
    const size_t tiles = 2 * WAVES * 32 * Tile<T, D>::NS * 16 + 4 * 32 * WAVES + PackedBias::bytes(g.a, g.pack);
    const size_t join = 4 * 64 * WAVES * (2 + D / 2), lds = tiles > join ? tiles : join;
    if (modified(g.a)) launch(mmt_long_attn_few_kernel<T, D, true>, g.items, lds, st, g);
    else launch(mmt_long_attn_few_kernel<T, D, false>, g.items, lds, st, g);
    return;
  }
  const size_t tiles = 4 * Tile<T, D>::BYTES + 8 * Tile<T, D>::BK, rest = 24 * WAVES + 4 * Lut::floats(g.a);
  if constexpr (sizeof(T) == 2) {
    if (g.teams == 2) {
      if (modified(g.a)) launch(mmt_long_attn_fwd_kernel<T, D, GAPS, true, 2>, g.items, 2 * tiles + rest, st, g, 2 * THREADS);
      else launch(mmt_long_attn_fwd_kernel<T, D, GAPS, false, 2>, g.items, 2 * tiles + rest, st, g, 2 * THREADS);
      return;
    }
  }
  if (modified(g.a)) launch(mmt_long_attn_fwd_kernel<T, D, GAPS, true, 1>, g.items, tiles + rest, st, g);
  else launch(mmt_long_attn_fwd_kernel<T, D, GAPS, false, 1>, g.items, tiles + rest, st, g);
}

template <typename T, int D, bool GAPS, int TEAMS> static void dq_launch(const Args &g, int64_t items, hipStream_t st) {
  const size_t lds = TEAMS * (4 * Tile<T, D>::BYTES + 8 * Tile<T, D>::BK) + 24 * WAVES + 4 * Lut::floats(g.a);
  if (modified(g.a)) launch(mmt_long_attn_dq_kernel<T, D, GAPS, true, TEAMS>, items, lds, st, g, TEAMS * THREADS);
  else launch(mmt_long_attn_dq_kernel<T, D, GAPS, false, TEAMS>, items, lds, st, g, TEAMS * THREADS);
}

template <typename T, int D, bool GAPS> static void bwd_size(Args &g, hipStream_t st, float *table_part, float *dtable) {
  typedef Tile<T, D> L;
  const mmt_long_attention &a = g.a;
  const bool mod = modified(a);
  const size_t small = 24 * WAVES;
  const int64_t qitems = (int64_t)a.B * a.H * g.nqt;
  if constexpr (sizeof(T) == 2) {
    if (g.teams == 2) dq_launch<T, D, GAPS, 2>(g, qitems, st);
    else dq_launch<T, D, GAPS, 1>(g, qitems, st);
  } else {
    dq_launch<T, D, GAPS, 1>(g, qitems, st);
  }
  if (a.rel_bias) {
    const size_t lds = 2 * L::BYTES + 8 * L::BK + small + 4 * Lut::floats(a) + ((Lut::floats(a) + 15) & ~15) + (size_t)WAVES * a.n_buckets * 256;
    (void)hipFuncSetAttribute((const void *)mmt_long_attn_table_kernel<T, D>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL((mmt_long_attn_table_kernel<T, D>), dim3((unsigned)qitems), dim3(THREADS), lds, st, g, table_part);
    hipLaunchKernelGGL(mmt_long_attn_table_sum_kernel<T>, dim3(a.H * a.n_buckets), dim3(64), 0, st, a, (int64_t)a.B * g.nqt, table_part,
                       g.far_part, dtable);
  }
  const size_t lds_k = 4 * L::BYTES + 24 * L::BK + small + 4 * Lut::floats(a);
  const int64_t kitems = (int64_t)g.groups * ((a.Lk + ROWS - 1) / ROWS) * g.zh * g.zq;
  if constexpr (sizeof(T) == 2 && D > 64) {
    const size_t lds2 = 4 * L::BYTES + 2 * 128 * 64 * 2 + 24 * 64 + 80 + 4 * Lut::floats(a);
    if (mod) launch(mmt_long_attn_dkv2_kernel<T, D, GAPS, true>, kitems, lds2, st, g, 512);
    else launch(mmt_long_attn_dkv2_kernel<T, D, GAPS, false>, kitems, lds2, st, g, 512);
  } else {
    if (mod) launch(mmt_long_attn_dkv_kernel<T, D, GAPS, true>, kitems, lds_k, st, g);
    else launch(mmt_long_attn_dkv_kernel<T, D, GAPS, false>, kitems, lds_k, st, g);
  }
}

template <typename T> static void docs(const Args &g, DocRange *out, bool queries, hipStream_t st) {
  const int bk = Elem<T>::BK, nk = g.a.B * g.nkt, total = nk + (queries ? g.a.B * ((g.a.Lq + bk - 1) / bk) : 0);
  hipLaunchKernelGGL(mmt_long_attn_docs_kernel<T>, dim3((total + 3) / 4), dim3(256), 0, st, g, bk, nk, total, out);
}

// The instantiation of a head size: the next of 32, 64, 96, 128, and whether it leaves slots empty that have to be cleared (as a question
// of every step this cost the kernels 2 to 4 % at the head sizes that leave none)
template <typename F> static void by_size(int dh, F f) {
  if (dh < 32) f(Const<32>(), Const<1>());
  else if (dh == 32) f(Const<32>(), Const<0>());
  else if (dh < 64) f(Const<64>(), Const<1>());
  else if (dh == 64) f(Const<64>(), Const<0>());
  else if (dh < 96) f(Const<96>(), Const<1>());
  else if (dh == 96) f(Const<96>(), Const<0>());
  else if (dh < 128) f(Const<128>(), Const<1>());
  else f(Const<128>(), Const<0>());
}

template <typename T> void forward(Args &g, DocRange *ranges, hipStream_t st) {
  const mmt_long_attention &a = g.a;
  if (ranges && !g.few) docs<T>(g, ranges, false, st), g.krng = ranges;
  by_size(a.dh, [&](auto size, auto gaps) { fwd_size<T, decltype(size)::value, decltype(gaps)::value != 0>(g, st); });
  if (g.nsplit > 1) {
    const int64_t rows = (int64_t)a.B * a.H * a.Lq;
    hipLaunchKernelGGL(mmt_long_attn_join_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, g);
  }
}

template <typename T> void backward(Args &g, DocRange *ranges, f32x4 *maxima, float *table_part, float *dtable, hipStream_t st) {
  const mmt_long_attention &a = g.a;
  if (ranges) docs<T>(g, ranges, true, st), g.krng = ranges, g.qrng = ranges + (int64_t)a.B * g.nkt;
  if (maxima) {
    const int64_t rows = (int64_t)a.B * (a.Lq * (int64_t)a.H > a.Lk * (int64_t)a.Hk ? a.Lq * (int64_t)a.H : a.Lk * (int64_t)a.Hk), blocks = (rows + STAT_ROWS - 1) / STAT_ROWS;
    g.stat_parts = (int)(blocks < STAT_PARTS ? blocks : STAT_PARTS);
    g.maxima = maxima;
    g.dscale = (float *)(maxima + STAT_PARTS);
    hipLaunchKernelGGL(mmt_long_attn_maxima_kernel<T>, dim3(g.stat_parts), dim3(STAT_THREADS), 0, st, g, maxima);
  }
  by_size(a.dh, [&](auto size, auto gaps) { bwd_size<T, decltype(size)::value, decltype(gaps)::value != 0>(g, st, table_part, dtable); });
  if (g.part_dk) {
    const int64_t n = (int64_t)a.B * a.Lk * a.Hk * a.dh;
    hipLaunchKernelGGL(mmt_long_attn_dkv_sum_kernel<T>, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st, g);
  }
}

}  // namespace la
