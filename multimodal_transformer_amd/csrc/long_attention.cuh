// Device code shared by the long-sequence attention kernels (long_attention.hip): element types, LDS tiles, score transform.
//
// Mathematics.  For query i of a row of n keys (position p = n - Lq + i) and key j:
//   s = scale q_i . k_j;   u = cap tanh(s / cap);   u += -slope_h |p - j| + table[h][bucket(j - p)]
//   visible: j < n, equal documents, and (not causal, or j <= p, or j < prefix)   <=>   j < hi_i  and equal documents
//   P = softmax of u over the visible keys (0 where there is none);   o = P v
// Everything runs on v_mfma_f32_32x32x16 (16-bit types) or chains of v_mfma_f32_32x32x2 (fp32) with the SCORES TRANSPOSED: the
// key is the row and the query the column of the 32 x 32 accumulator, so that a lane owns ONE query (lane % 32) and 16 of 32 keys:
// row maximum and sum stay in the lane but for one exchange between the wave's halves, the rescaling factor is a lane's own scalar,
// and the 16 probabilities of a lane are, eight at a time, exactly the B operand of the next product (o^T += v^T P^T) when its
// reduction index runs over the keys in the accumulator's order.  P never leaves the registers.
//   C layout of a 32 x 32 tile: column = lane % 32, register i -> row 8 (i / 4) + 4 (lane / 32) + i % 4
//   A / B operands of a 16-deep step: row / column = lane % 32, element e of lane half h -> reduction index 8 h + e; any one-to-one
//   relabelling of that index is allowed as long as A and B share it: the second product uses
//   index (h, e) -> key 16 c + 4 h + e % 4 + 8 (e / 4), the order in which accumulator registers 8 c .. 8 c + 7 hold the keys.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "long_attention_args.cuh"

namespace la {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

template <int N> struct Const {
  static constexpr int value = N;
};

// ---- element types --------------------------------------------------------------------------------------------------------
// BK: keys (queries, in the key-gradient kernel) per LDS tile; fp32 elements are twice as large, so half as many.
// PSHIFT: probabilities are multiplied by 2^PSHIFT before they are rounded to the element type (and the sums with them): fp16 has
// 5 exponent bits, so that without it every probability under 2^-14 would lose digits and every one under 2^-25 vanish.
// SLACK: by so much, in units of log 2, a score may exceed what its exponential refers to; in fp16 2^(PSHIFT + SLACK) has to stay finite.
template <typename T> struct Elem;
template <> struct Elem<__bf16> {
  typedef bf16x8 V8;
  typedef bf16x4 V4;
  static constexpr int BK = 64;
  static constexpr float PSHIFT = 0.f, SLACK = 8.f;
  static __device__ __forceinline__ f32x16 mma(const V8 &a, const V8 &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Elem<_Float16> {
  typedef f16x8 V8;
  typedef f16x4 V4;
  static constexpr int BK = 64;
  static constexpr float PSHIFT = 14.f, SLACK = 1.f;
  static __device__ __forceinline__ f32x16 mma(const V8 &a, const V8 &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Elem<float> {
  typedef f32x8 V8;
  typedef f32x4 V4;
  static constexpr int BK = 32;
  static constexpr float PSHIFT = 0.f, SLACK = 8.f;
  // eight 2-deep steps; step e pairs element e of the two lane halves, which is what the 16-bit instruction sums too
  static __device__ __forceinline__ f32x16 mma(const V8 &a, const V8 &b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

template <typename T> __device__ __forceinline__ typename Elem<T>::V8 round8(const float *x) {   // round to nearest even
  typename Elem<T>::V8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (T)x[e];
  return r;
}

// The thread index where nothing derived from it may be taken for loop invariant: in the paths that few tiles take (masks, ragged ends),
// what the compiler computes ahead of the loop would occupy registers in all of it.
__device__ __forceinline__ int rare_tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// ---- LDS tiles ------------------------------------------------------------------------------------------------------------
// BK rows of D elements in 16-byte slots, NS slots per row (a power of two, so that a slot's place is an exclusive or).  A row
// operand reads one slot of 32 different rows, a transposed read (ds_read_b64_tr_b16: four rows x 16 columns per 16 lanes) four
// consecutive rows x four consecutive slots: the exclusive or spreads both over the 64 banks (16 slots).
template <typename T, int D> struct Tile {
  static constexpr int EPS = 16 / (int)sizeof(T);                 // elements per slot
  static constexpr int DS = D <= 32 ? 32 : D <= 64 ? 64 : 128;
  static constexpr int NS = DS / EPS;
  static constexpr int BK = Elem<T>::BK;
  static constexpr int BYTES = BK * NS * 16;
  static constexpr int PERIOD = sizeof(T) == 4 ? (NS == 8 ? 16 : 8) : 16;     // swz depends on row % PERIOD
  static __device__ __forceinline__ int swz(int row, int slot) {
    if constexpr (sizeof(T) == 4) {
      return slot ^ (NS >= 16 ? (row & 7) : ((row >> 1) & 7));
    } else {
      if constexpr (NS == 16) return slot ^ (((row & 3) << 2) | ((row >> 2) & 3));
      else if constexpr (NS == 8) return slot ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
      else return slot ^ ((row >> 2) & 3);
    }
  }
};
// row operand: elements 16 c + 8 h .. + 7 of row `row`
template <typename T, int D> __device__ __forceinline__ typename Elem<T>::V8 row_frag(const char *t, int row, int c, int h) {
  typedef Tile<T, D> L;
  if constexpr (sizeof(T) == 2) {
    return *(const typename Elem<T>::V8 *)(t + (row * L::NS + L::swz(row, 2 * c + h)) * 16);
  } else {
    const f32x4 a = *(const f32x4 *)(t + (row * L::NS + L::swz(row, 4 * c + 2 * h)) * 16);
    const f32x4 b = *(const f32x4 *)(t + (row * L::NS + L::swz(row, 4 * c + 2 * h + 1)) * 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// transposed operand: column 32 dt + lane % 32 of rows r0 + 4 h + {0..3} and r0 + 8 + 4 h + {0..3}
template <typename T, int D> __device__ __forceinline__ typename Elem<T>::V8 col_frag(const char *t, int r0, int dt, int lane) {
  typedef Tile<T, D> L;
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    // lane i of a group of 16 hands in row i / 4, columns 4 (i % 4) .. + 3 and receives column i of the four rows
    const int i = lane & 15, col = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
    s16x4 p[2];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int row = r0 + 8 * part + 4 * h + (i >> 2);
      const char *a = t + (row * L::NS + L::swz(row, col >> 3)) * 16 + (col & 7) * 2;
      p[part] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)a);
    }
    return __builtin_bit_cast(typename Elem<T>::V8, __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const int col = 32 * dt + (lane & 31);
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int row = r0 + 8 * (e >> 2) + 4 * h + (e & 3);
      r[e] = *(const float *)(t + (row * L::NS + L::swz(row, col >> 2)) * 16 + (col & 3) * 4);
    }
    return r;
  }
}

// Row operand straight from memory (the tile that stays in registers), whatever the row holds: requested before it is known which rows
// are live, so that a workgroup's first loads wait for nothing.  `live_frag` zeroes dead rows, and elements at and beyond dh, and is where
// the operand has to be here.
template <typename T> __device__ __forceinline__ typename Elem<T>::V8 mem_frag(const T *row, int c, int h, int dh) {
  const int d = 16 * c + 8 * h;
  return *(const typename Elem<T>::V8 *)(row + (d < dh ? d : 0));
}
template <typename V> __device__ __forceinline__ void live_frag(V &v, int c, int h, int dh, bool live) {
  const bool in = live && 16 * c + 8 * h < dh;
  v = in ? v : V{};
  asm volatile("" : "+v"(v));
}
// a value that all lanes share and that this kernel does not write
template <typename V> __device__ __forceinline__ V scalar_load(const V *p) { return *(const __attribute__((address_space(4))) V *)(uintptr_t)p; }

// What was loaded ahead of a loop has arrived here (live_frag does the same).  Otherwise the compiler waits for it at its first use inside the loop, every time
// around - and with it, requests being counted in order, for the tile that has just been asked for.
template <typename V> __device__ __forceinline__ void settle(V &v) { asm volatile("" : "+v"(v)); }

// One 16-byte piece per lane straight from memory into LDS (no registers in between): lane l's piece lands at lds + 16 l.
// Untracked by the compiler: dma_wait before the barrier that publishes the tile.  M0 holds the LDS address.
__device__ __forceinline__ void dma16(const void *base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory");
}
// all but the newest N requests of the wave have arrived (requests of the compiler's own in between only make this stricter)
template <int N> __device__ __forceinline__ void dma_wait() {
  static_assert(N == 0 || N == 2 || N == 4 || N == 8 || N == 16, "one of the tiles' request counts");
  if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  else if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2)" : : : "memory");
  else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" : : : "memory");
  else if constexpr (N == 8) asm volatile("s_waitcnt vmcnt(8)" : : : "memory");
  else asm volatile("s_waitcnt vmcnt(16)" : : : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void *p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char *)p;
}

// Tiles of a (rows, dh) matrix on their way to LDS.  A lane's byte offset inside a tile is the same for every tile; the tile's own
// part is a scalar.  Slots at and beyond dh repeat slot 0 and rows at and beyond n_rows the last row (nothing outside the tensor is
// read); their results are masked or nobody stores them, but for row operands, where the slots beyond dh meet zeros (0 x inf is not 0):
// `clear_pads` makes them zero.
// NT threads (the workgroup, or one wave) move tiles of R rows, NT / NS rows at a time; where the exclusive or of a row repeats after
// as many rows, the steps differ by a scalar and one offset serves them all.
template <typename T, int D, int R = Tile<T, D>::BK, int NT = THREADS> struct Dma {
  typedef Tile<T, D> L;
  static constexpr int N = R * L::NS / NT, STEP = NT / L::NS;
  static constexpr bool ONE = STEP % L::PERIOD == 0;
  static_assert(N * NT == R * L::NS && STEP * L::NS == NT, "a tile is a whole number of 16-byte loads per thread");
  const char *base;
  int64_t rs;                        // bytes between rows; 64 rows stay below 2^31 bytes
  int n_rows;
  unsigned off[ONE ? 1 : N];
  __device__ __forceinline__ void init(const T *p, int64_t row_stride, int rows, int dh) {
    base = (const char *)p, rs = row_stride * (int64_t)sizeof(T), n_rows = rows;
#pragma unroll
    for (int n = 0; n < (ONE ? 1 : N); ++n) {
      const int idx = threadIdx.x % NT + n * NT, row = idx / L::NS, slot = L::swz(row, idx % L::NS);
      off[n] = (unsigned)((ONE ? row : row - n * STEP) * rs) + (slot * L::EPS < dh ? slot * 16 : 0);
    }
  }
  __device__ __forceinline__ void load(unsigned lds, int r0) const {
    const char *b = base + r0 * rs;
    const unsigned mine = __builtin_amdgcn_readfirstlane(lds + ((threadIdx.x % NT) >> 6) * 1024);
    if (r0 + R <= n_rows) {
#pragma unroll
      for (int n = 0; n < N; ++n) dma16(b + n * STEP * rs, off[ONE ? 0 : n], mine + n * NT * 16);
    } else {
      // the rows beyond the last one repeat it
      const int first = (rare_tid() % NT) / L::NS;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int row = first + n * STEP, over = max(0, r0 + row - (n_rows - 1));
        dma16(b, off[ONE ? 0 : n] + (unsigned)(n * STEP * rs) - (unsigned)(over * rs), mine + n * NT * 16);
      }
    }
  }
  // The tile's own requests have arrived (dma_wait): each lane clears those of its pieces that lie beyond dh, ahead of the barrier that
  // publishes the tile.  Only half of a chunk of 16 elements: chunks wholly beyond dh are not read (has_chunk).
  static __device__ __forceinline__ void clear_pads(char *tile, int dh) {
    if (dh % 16 == 0) return;
    const int tid = rare_tid() % NT;
    auto beyond = [&](int idx) {
      const int d = L::swz(idx / L::NS, idx % L::NS) * L::EPS;
      return d >= dh && d < dh + 8;
    };
    if constexpr (ONE) {
      if (!beyond(tid)) return;
#pragma unroll
      for (int n = 0; n < N; ++n) *(u32x4 *)(tile + (tid + n * NT) * 16) = u32x4{};
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (beyond(tid + n * NT)) *(u32x4 *)(tile + (tid + n * NT) * 16) = u32x4{};
    }
  }
};

// Whether chunk c of an operand's 16 elements holds any of the head's: where dh leaves slots empty (GAPS) the last chunk may not
template <bool GAPS, int NC> __device__ __forceinline__ bool has_chunk(int c, int dh) { return !GAPS || c < NC - 1 || 16 * c < dh; }

// Rows of a tile that must not take part become zeros (whatever they hold: 0 x NaN would reach every other row): at and beyond `end`
// (tile row), or with a negative document id
template <typename T, int D, int R = Tile<T, D>::BK, int NT = THREADS>
__device__ __forceinline__ void zero_rows(char *lds, int end, const int *doc) {
  typedef Tile<T, D> L;
  const int tid = rare_tid() % NT;
#pragma unroll
  for (int n = 0; n < R * L::NS / NT; ++n) {
    const int idx = tid + n * NT, row = idx / L::NS;
    if (row >= end || (doc && doc[row] < 0)) *(u32x4 *)(lds + idx * 16) = u32x4{};
  }
}

// ---- lanes ----------------------------------------------------------------------------------------------------------------
// the two halves of the wave hold complementary parts of a row: v[lane] op v[lane ^ 32]
// (s_nop: the distance from a VALU write to the lane swap, which the compiler does not see inside asm)
__device__ __forceinline__ float half_max(float v) {
  float a = v, b = v;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float v) {
  float a = v, b = v;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return a + b;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = min(v, __shfl_xor(v, m));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = max(v, __shfl_xor(v, m));
  return __builtin_amdgcn_readfirstlane(v);
}
// what the wave has read from and written to LDS so far is done before what follows, requests straight into LDS among it
__device__ __forceinline__ void wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ int acc_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }
// a number per accumulator row of a lane, from 32 in LDS (16-byte aligned)
__device__ __forceinline__ void acc_rows(f32x4 *v, const float *s, int h) {
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] = *(const f32x4 *)(s + 8 * q + 4 * h);
}

// ---- score transform ------------------------------------------------------------------------------------------------------
// tanh without cancellation.  |y| <= 3/8: odd series to y^11, remainder < 21844/6081075 y^13 = 3e-8 of y; over all floats of that range it
// is off by at most 7.5e-8 of the value.  Beyond: 1 - 2 / (1 + e^2y).  With an ulp each of the exponential and the reciprocal, and the
// roundings of the argument and the sums, arithmetic allows 6.3e-7 of the value at 3/8; over all floats up to 10 it is at most 2.3e-7 (at
// 0.552), and falls off from there.
__device__ __forceinline__ float tanh_series(float y) {
  const float z = y * y;
  float p = fmaf(z, -8.86323552990219657e-3f, 2.18694885361552028e-2f);
  p = fmaf(z, p, -5.39682539682539683e-2f);
  p = fmaf(z, p, 1.33333333333333333e-1f);
  p = fmaf(z, p, -3.33333333333333333e-1f);
  return fmaf(y * z, p, y);
}
__device__ __forceinline__ float tanh_any(float y) {
  asm volatile("" : "+v"(y));                             // (or the series, common to both ways, is hoisted for all elements at once)
  const float e = ex2(y * (2.f * LOG2E));
  float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e), small = tanh_series(y);
  asm volatile("" : "+v"(big), "+v"(small));              // (both are computed: a branch per element costs more)
  return fabsf(y) <= 0.375f ? small : big;
}
// x -> tanh(x * f) for N scores of a lane; most tiles of a trained model stay inside the series' range: one wave-uniform branch
template <int N> __device__ __forceinline__ void tanh_scores(float *x, float f) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] *= f;
    m = fmaxf(m, fabsf(x[i]));
  }
  if (__any(!(m <= 0.375f))) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = tanh_any(x[i]);
      if (i % 2) __builtin_amdgcn_sched_barrier(0);       // (two at a time: all at once would set the kernel's register count)
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = tanh_series(x[i]);
  }
}

// ---- work distribution ----------------------------------------------------------------------------------------------------
// Workgroups go round-robin over the 8 XCDs, each with its own L2.  Item n belongs to group n % groups (the workgroups that read the
// same keys and values): with a multiple of 8 groups each stays on one XCD, and within all groups the items come in the order
// n / groups, the longest first.

// tiles t0 <= t < t1 whose documents overlap [lo, hi], in order; 64 tiles are looked up at a time, one per lane
struct TileIter {
  const DocRange *rng;
  int lo, hi, base, end;
  unsigned long long mask;
  DocRange mine;
  int cur_lo, cur_hi, cur_dead;                      // of the tile that next() returned
  // `ready`: the ranges of tiles t0 .. t0 + 63, one per lane, where they have been loaded already
  static __device__ __forceinline__ DocRange ahead(const DocRange *r, int t0, int n_tiles) {
    return r ? r[min(t0 + (int)(threadIdx.x & 63), n_tiles - 1)] : DocRange{0, 0, 0, 0};
  }
  __device__ __forceinline__ void start(const DocRange *r, int l, int h, int t0, int t1, DocRange ready) {
    rng = r, lo = l, hi = h, base = t0, end = t1;
    mine = ready;
    cur_lo = cur_hi = cur_dead = 0;
    mask = __ballot(base + (int)(threadIdx.x & 63) < end && (!rng || (mine.lo <= hi && mine.hi >= lo)));
  }
  __device__ __forceinline__ void here() { settle(mine.lo), settle(mine.hi), settle(mine.dead); }     // (ahead of a loop: see settle)
  __device__ __forceinline__ void fill() {
    const int t = base + (threadIdx.x & 63);
    bool ok = t < end;
    if (ok && rng) {
      mine = rng[t];
      ok = mine.lo <= hi && mine.hi >= lo;
    }
    mask = __ballot(ok);
  }
  __device__ __forceinline__ int next() {            // -1 when there is none left
    while (mask == 0) {
      base += 64;
      if (base >= end) return -1;
      fill();
    }
    const int n = __builtin_ctzll(mask);
    mask &= mask - 1;
    if (rng) {
      cur_lo = __builtin_amdgcn_readlane(mine.lo, n);
      cur_hi = __builtin_amdgcn_readlane(mine.hi, n);
      cur_dead = __builtin_amdgcn_readlane(mine.dead, n);
    }
    return __builtin_amdgcn_readfirstlane(base + n);
  }
  // at most `most` tiles are left, those that have not been looked up yet among them (256 at a time: one wait for memory)
  __device__ __forceinline__ bool at_most(int most) const {
    int n = __popcll(mask);
    for (int t0 = base + 64; n <= most && t0 < end; t0 += 256) {
      if (!rng) return false;                            // (a whole lookup, and more behind it)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = t0 + 64 * u + (int)(threadIdx.x & 63);
        const DocRange r = rng[min(t, end - 1)];
        n += __popcll(__ballot(t < end && r.lo <= hi && r.hi >= lo));
      }
    }
    return n <= most;
  }
  // not a single document that all rows of [lo, hi] share: masks are needed
  __device__ __forceinline__ bool mixed() const { return rng && !(cur_dead == 0 && cur_lo == cur_hi && lo == hi && lo == cur_lo); }
};

// The tiles of an iterator dealt to the teams of a workgroup, one each at a time.  All of it is the same in all waves but for what is
// this team's: its tile (-1: none this time), whether that needs document masks, whether it holds rows that have to be zeroed.
template <int TEAMS> struct Deal {
  TileIter it;
  int lead, t;                       // the first team's tile: -1 ends the loop for all
  bool mixed, zero, any_zero;        // any_zero: some team zeroes rows, all meet once more
  __device__ __forceinline__ bool zeroes(int tile, int bk, int len) const { return tile * bk + bk > len || (it.mixed() && it.cur_dead != 0); }
  __device__ __forceinline__ void next(int team, int bk, int len) {
    lead = t = it.next();
    mixed = it.mixed(), any_zero = zero = zeroes(t, bk, len);
    if constexpr (TEAMS == 2) {
      if (lead < 0) return;
      const int other = it.next();
      const bool z = other >= 0 && zeroes(other, bk, len);
      any_zero = zero || z;
      if (team) t = other, mixed = it.mixed(), zero = z;
    }
  }
};

}  // namespace la
