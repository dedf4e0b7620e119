// Norm of queries and keys per head + rotation of their positions in one pass over memory (mmt_qk_norm_rope_fwd / _bwd).
//
// A group of LPH lanes (the power of two at or above dh / 8) holds one head of one token, 8 elements per lane: the mean square and,
// backwards, the dot product are reductions inside the group, everything else stays in the lane; with the half-split pairing a
// pair's other element comes from the lane rot / 16 further on.  Both go through the VALU's lane crossings (DPP), not through LDS.
// The angles of a token are shared by all its heads: a workgroup forms them once per token, in 64 bits (position * frequency reaches
// 10^6 turns, of which fp32 would keep 2 digits), reduces them to a fraction of a turn, and a lane keeps the cosines and sines of its 8
// elements in registers while it walks over the token's heads.  Bound by memory: every element is read once and written once
// (backwards: two read, one written).  bf16, 4 x 4096 tokens x 20 heads of 128: 39 us forward, 4.3 TB/s, 64 us backward, 3.9 TB/s, and 6 for the
// sum of the weights' gradients, where a large copy reaches 4.9.  32 single tokens of 20 heads: 6 us, the launch and three waits for memory.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mmt_amd.h"
#include "mmt_gfx950.cuh"

int mmt_set_error(int code, const char *fmt, ...);   // transformer.hip

namespace {

constexpr int NT = 256;
// workgroups backwards, each with a part of the weights' gradients: half as many take a tenth longer in the case above, and their sum 4 us instead of 6
constexpr int MAX_PARTS = 2048;

template <typename T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

template <typename T> __device__ __forceinline__ void widen(const typename Vec8<T>::type &v, float *x) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float *x) {
  typename Vec8<T>::type v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)x[e];
  *(typename Vec8<T>::type *)p = v;
}
template <typename T> __device__ __forceinline__ float weight_at(const void *w, int w_f32, int d) {
  return w_f32 ? ((const float *)w)[d] : (float)((const T *)w)[d];
}

struct Grads {
  const void *dqo, *dko;
  int64_t q_bs, q_rs, q_hs, k_bs, k_rs, k_hs;
  void *dq, *dk;
  float *part;               // (workgroups, 2, dh)
};

// cosine and sine of the angles of tokens t0 .. t0 + tok - 1 -> cs[token][pair]
__device__ __forceinline__ void angles(const mmt_qk_norm_rope &a, int64_t t0, int tok, float2 *cs) {
  const int half = a.rot / 2;
  for (int n = threadIdx.x; n < tok * half; n += NT) {
    const int64_t t = t0 + n / half;
    const double pos = a.positions ? (double)a.positions[t] : (double)(t % a.L);
    const double turns = pos * (a.inv_freq[n % half] * 0.15915494309189533577);      // 1 / (2 pi)
    float s, c;
    sincospif((float)(2. * (turns - rint(turns))), &s, &c);
    cs[n] = make_float2(c, s);
  }
}

// sum over the LPH lanes of a group, in all of them
template <int LPH> __device__ __forceinline__ float group_sum(float v) {
  v += dpp_mov<0xB1>(v);                                // quad_perm: lane ^ 1, lane ^ 2
  v += dpp_mov<0x4E>(v);
  if (LPH >= 8) v += dpp_mov<0x141>(v);                 // row_half_mirror
  if (LPH >= 16) v += dpp_mov<0x140>(v);                // row_mirror
  if (LPH == 32) v += __shfl_xor(v, 16);
  return v;
}
// v of lane ^ S
template <int S> __device__ __forceinline__ float lane_xor(float v) {
  if constexpr (S == 1) return dpp_mov<0xB1>(v);
  else if constexpr (S == 2) return dpp_mov<0x4E>(v);
  else if constexpr (S == 8) return dpp_mov<0x128>(v);  // row_ror:8
  else if constexpr (S == 4) {                          // row_shl:4 into the lower four lanes of each eight, row_shr:4 into the upper
    const int i = __builtin_bit_cast(int, v);
    const int low = __builtin_amdgcn_update_dpp(0, i, 0x104, 0xF, 0x5, false);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(low, i, 0x114, 0xF, 0xA, false));
  } else return __shfl_xor(v, S);
}
// the pair partners of a lane's 8 elements with the half-split pairing and halves of whole lanes (half / 8 of them)
template <int LPH> __device__ __forceinline__ void partners(const float *v, float *o, int lane_in, int step) {
#define MMT_PARTNERS(S)                                 \
  if (LPH >= 2 * S && step == S) {                      \
    _Pragma("unroll") for (int e = 0; e < 8; ++e) o[e] = lane_xor<S>(v[e]); \
    return;                                             \
  }
  MMT_PARTNERS(1) MMT_PARTNERS(2) MMT_PARTNERS(4) MMT_PARTNERS(8) MMT_PARTNERS(16)
#undef MMT_PARTNERS
  const int src = (threadIdx.x & 63) - lane_in + ((lane_in < step ? lane_in + step : lane_in - step) & (LPH - 1));
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = __shfl(v[e], src);
}

// tok tokens per step and workgroup, their heads dealt over split lane groups each (tok * split = groups of the workgroup)
template <typename T, int LPH, bool BWD> __global__ void __launch_bounds__(NT) mmt_qk_norm_rope_kernel(const mmt_qk_norm_rope a, const Grads g, void *q_out, void *k_out, int split) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef typename Vec8<T>::type V8;
  constexpr int GROUPS = NT / LPH;
  float2 *cs = (float2 *)smem;
  const int lane_in = threadIdx.x % LPH, group = threadIdx.x / LPH, d0 = lane_in * 8, half = a.rot / 2, heads = a.H + a.Hk;
  const int tok = GROUPS / split, lt = group / split, h0 = group % split;
  const float inv_dh = 1.f / (float)a.dh;
  const bool on = d0 < a.dh, by_lane = half % 8 == 0;
  const int64_t tokens = (int64_t)a.B * a.L;
  float wq[8], wk[8], sq[8] = {}, sk[8] = {};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wq[e] = on ? weight_at<T>(a.q_weight, a.w_dtype == MMT_F32, d0 + e) : 0.f;
    wk[e] = on ? weight_at<T>(a.k_weight, a.w_dtype == MMT_F32, d0 + e) : 0.f;
  }
  for (int64_t t0 = (int64_t)blockIdx.x * tok; t0 < tokens; t0 += (int64_t)gridDim.x * tok) {
    const int nt = (int)min((int64_t)tok, tokens - t0);
    const int64_t t = t0 + (lt < nt ? lt : 0), b = t / a.L, i = t - b * a.L;
    const bool mine = lt < nt && on;
    const T *qrow = (const T *)a.q + b * a.q_bs + i * a.q_rs, *krow = (const T *)a.k + b * a.k_bs + i * a.k_rs - a.H * a.k_hs;
    const T *qgrad = BWD ? (const T *)g.dqo + b * g.q_bs + i * g.q_rs : nullptr, *kgrad = BWD ? (const T *)g.dko + b * g.k_bs + i * g.k_rs - a.H * g.k_hs : nullptr;
    V8 next = {}, gnext = {};
    auto fetch = [&](int hh) {                          // (one head ahead)
      const bool is_k = hh >= a.H;
      next = *(const V8 *)((is_k ? krow + hh * a.k_hs : qrow + hh * a.q_hs) + d0);
      if (BWD) gnext = *(const V8 *)((is_k ? kgrad + hh * g.k_hs : qgrad + hh * g.q_hs) + d0);
    };
    if (mine && h0 < heads) fetch(h0);
    __syncthreads();
    angles(a, t0, nt, cs);
    __syncthreads();
    float c[8], sn[8];                                  // y = v c + partner sn; elements that are not turned: 1, 0
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      const bool first = a.interleaved ? !(d & 1) : d < half, turned = d < a.rot && lt < nt;
      const float2 v = turned ? cs[lt * half + (a.interleaved ? d >> 1 : first ? d : d - half)] : make_float2(1.f, 0.f);
      c[e] = v.x;
      sn[e] = first != BWD ? -v.y : v.y;                // forward: (-, +) for (first, second); the gradient turns back
    }
    for (int hh = h0; hh < heads; hh += split) {
      const bool is_k = hh >= a.H;
      float x[8], gy[8];
      widen<T>(next, x);
      if (BWD) widen<T>(gnext, gy);
      if (mine && hh + split < heads) fetch(hh + split);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
      const float r = 1.f / sqrtf(group_sum<LPH>(ss) * inv_dh + a.eps);
      float v[8], o[8];                                 // what is turned (forward: the norm, backward: the gradient), and its partners
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = BWD ? gy[e] : x[e] * r * (is_k ? wk[e] : wq[e]);
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e ^ 1];
      } else if (by_lane) {
        partners<LPH>(v, o, lane_in, half / 8);
      } else {                                          // a half ends inside a lane: element by element from memory
        const void *wrow = is_k ? a.k_weight : a.q_weight;
        const T *row = BWD ? (is_k ? kgrad + hh * g.k_hs : qgrad + hh * g.q_hs) : (is_k ? krow + hh * a.k_hs : qrow + hh * a.q_hs);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = d0 + e, p = d < half ? d + half : d - half;
          o[e] = 0.f;
          if (mine && d < a.rot) o[e] = BWD ? (float)row[p] : (float)row[p] * r * weight_at<T>(wrow, a.w_dtype == MMT_F32, p);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = d0 + e < a.rot ? fmaf(o[e], sn[e], v[e] * c[e]) : v[e];
      T *out;
      if (!BWD) {
        out = is_k ? (T *)k_out + (t * a.Hk + (hh - a.H)) * a.dh : (T *)q_out + (t * a.H + hh) * a.dh;
      } else {
        out = is_k ? (T *)g.dk + (t * a.Hk + (hh - a.H)) * a.dh : (T *)g.dq + (t * a.H + hh) * a.dh;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = mine ? v[e] * x[e] * r : 0.f;
          if (is_k) sk[e] += u;
          else sq[e] += u;
          v[e] *= is_k ? wk[e] : wq[e];
          dot = fmaf(v[e], x[e], dot);
        }
        const float f = group_sum<LPH>(dot) * r * r * inv_dh;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r * fmaf(-f, x[e], v[e]);
      }
      if (mine) store8(out + d0, v);
    }
  }
  if (BWD) {
    // the groups of the workgroup in order, then one part per workgroup
    float *s = (float *)smem;                // [group][LPH * 8]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) s[group * LPH * 8 + d0 + e] = which ? sk[e] : sq[e];
      __syncthreads();
      for (int d = threadIdx.x; d < a.dh; d += NT) {
        float v = 0.f;
        for (int u = 0; u < GROUPS; ++u) v += s[u * LPH * 8 + d];
        g.part[((int64_t)blockIdx.x * 2 + which) * a.dh + d] = v;
      }
    }
  }
}

// parts -> weight gradients, in 64 bits and in a fixed order: 64 threads per element, 16 neighbouring elements per workgroup
template <typename T> __global__ void __launch_bounds__(1024) mmt_qk_weight_sum_kernel(const float *part, int parts, int dh, int w_f32, void *dqw, void *dkw) {
  const int n = blockIdx.x * 16 + (threadIdx.x & 15), s = threadIdx.x >> 4;
  double v = 0.;
  if (n < 2 * dh) {
#pragma unroll 8
    for (int p = s; p < parts; p += 64) v += part[(int64_t)p * 2 * dh + n];
  }
  __shared__ double sum[64][17];
  sum[s][threadIdx.x & 15] = v;
  __syncthreads();
  if (threadIdx.x >= 16 || n >= 2 * dh) return;
  v = 0.;
  for (int p = 0; p < 64; ++p) v += sum[p][threadIdx.x];
  void *w = n < dh ? dqw : dkw;
  const int d = n < dh ? n : n - dh;
  if (w_f32) ((float *)w)[d] = (float)v;
  else ((T *)w)[d] = (T)(float)v;
}

int check(const mmt_qk_norm_rope *a, const char *who) {
  if (!a || !a->q || !a->k || !a->q_weight || !a->k_weight || !a->inv_freq) return mmt_set_error(MMT_EINVAL, "%s: null pointer", who);
  if (a->dtype != MMT_F32 && a->dtype != MMT_BF16 && a->dtype != MMT_F16) return mmt_set_error(MMT_EINVAL, "%s: unknown element type %d", who, a->dtype);
  if (a->w_dtype != MMT_F32 && a->w_dtype != a->dtype) return mmt_set_error(MMT_EINVAL, "%s: weights are fp32 or of the tensors' type", who);
  if (a->B <= 0 || a->L <= 0 || a->H <= 0 || a->Hk <= 0) return mmt_set_error(MMT_EINVAL, "%s: B, L, H and Hk have to be positive", who);
  if (a->dh < 8 || a->dh > 256 || a->dh % 8) return mmt_set_error(MMT_EINVAL, "%s: head size %d, need a multiple of 8 up to 256", who, a->dh);
  if (a->rot < 2 || a->rot % 2 || a->rot > a->dh) return mmt_set_error(MMT_EINVAL, "%s: %d turned elements, need an even number up to the head size", who, a->rot);
  if (!(a->eps >= 0.f) || !isfinite(a->eps)) return mmt_set_error(MMT_EINVAL, "%s: eps has to be finite and not negative", who);
  if ((double)a->H + a->Hk > 65536. || (double)a->B * a->L > 2e9) return mmt_set_error(MMT_EINVAL, "%s: too many rows for one call", who);
  const int64_t unit = a->dtype == MMT_F32 ? 4 : 8;
  if (((uintptr_t)a->q | (uintptr_t)a->k) & 15 || (a->q_bs | a->q_rs | a->q_hs | a->k_bs | a->k_rs | a->k_hs) % unit)
    return mmt_set_error(MMT_EINVAL, "%s: rows of q and k have to start at multiples of 16 bytes", who);
  return MMT_OK;
}

// lane groups per token: one, unless there are too few tokens for 2048 workgroups that way (more than there are heads is no use); always
// one takes 18 us instead of 6 for 32 tokens of 20 heads of 128, 14 and 17 instead of 8 and 12 for 3111 of 16 heads of 32 in fp32
int lanes_per_head(const mmt_qk_norm_rope *a) { return a->dh <= 32 ? 4 : a->dh <= 64 ? 8 : a->dh <= 128 ? 16 : 32; }
int groups_per_token(const mmt_qk_norm_rope *a) {
  const int groups = NT / lanes_per_head(a);
  int split = 1;
  while (split < groups && split < a->H + a->Hk && (int64_t)a->B * a->L * split < (int64_t)2048 * groups) split *= 2;
  return split;
}
int tokens_per_group(const mmt_qk_norm_rope *a) { return NT / lanes_per_head(a) / groups_per_token(a); }
int workgroups(const mmt_qk_norm_rope *a, bool bwd) {
  const int tok = tokens_per_group(a);
  const int64_t n = ((int64_t)a->B * a->L + tok - 1) / tok;
  return (int)std::min<int64_t>(n, bwd ? MAX_PARTS : 16384);
}

template <typename T, int LPH, bool BWD>
void go(const mmt_qk_norm_rope *a, const Grads &g, void *qo, void *ko, hipStream_t st) {
  const int tok = tokens_per_group(a);
  size_t lds = (size_t)tok * (a->rot / 2) * sizeof(float2);
  if (BWD) lds = std::max(lds, (size_t)NT * 8 * sizeof(float));
  hipLaunchKernelGGL((mmt_qk_norm_rope_kernel<T, LPH, BWD>), dim3(workgroups(a, BWD)), dim3(NT), lds, st, *a, g, qo, ko, groups_per_token(a));
}
template <typename T, bool BWD> void by_size(const mmt_qk_norm_rope *a, const Grads &g, void *qo, void *ko, hipStream_t st) {
  const int lanes = lanes_per_head(a);
  if (lanes == 4) go<T, 4, BWD>(a, g, qo, ko, st);
  else if (lanes == 8) go<T, 8, BWD>(a, g, qo, ko, st);
  else if (lanes == 16) go<T, 16, BWD>(a, g, qo, ko, st);
  else go<T, 32, BWD>(a, g, qo, ko, st);
}
template <bool BWD> void by_type(const mmt_qk_norm_rope *a, const Grads &g, void *qo, void *ko, hipStream_t st) {
  if (a->dtype == MMT_BF16) by_size<__bf16, BWD>(a, g, qo, ko, st);
  else if (a->dtype == MMT_F16) by_size<_Float16, BWD>(a, g, qo, ko, st);
  else by_size<float, BWD>(a, g, qo, ko, st);
}

int status(const char *who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MMT_OK : mmt_set_error(MMT_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}

}  // namespace

extern "C" int mmt_qk_norm_rope_fwd(const mmt_qk_norm_rope *a, void *q_out, void *k_out, void *stream) {
  if (int rc = check(a, "mmt_qk_norm_rope_fwd")) return rc;
  if (!q_out || !k_out || ((uintptr_t)q_out | (uintptr_t)k_out) & 15) return mmt_set_error(MMT_EINVAL, "mmt_qk_norm_rope_fwd: outputs have to be 16-byte aligned addresses");
  by_type<false>(a, Grads{}, q_out, k_out, (hipStream_t)stream);
  return status("mmt_qk_norm_rope_fwd");
}

extern "C" size_t mmt_qk_norm_rope_workspace_bytes(const mmt_qk_norm_rope *a) {
  if (check(a, "mmt_qk_norm_rope_workspace_bytes")) return 0;
  return (size_t)workgroups(a, true) * 2 * a->dh * sizeof(float);
}

extern "C" int mmt_qk_norm_rope_bwd(const mmt_qk_norm_rope *a, const void *dqo, int64_t dq_bs, int64_t dq_rs, int64_t dq_hs, const void *dko,
                                    int64_t dk_bs, int64_t dk_rs, int64_t dk_hs, void *dq, void *dk, void *dq_weight, void *dk_weight,
                                    void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = check(a, "mmt_qk_norm_rope_bwd")) return rc;
  if (!dqo || !dko || !dq || !dk || !dq_weight || !dk_weight) return mmt_set_error(MMT_EINVAL, "mmt_qk_norm_rope_bwd: null pointer");
  const int64_t unit = a->dtype == MMT_F32 ? 4 : 8;
  if (((uintptr_t)dqo | (uintptr_t)dko | (uintptr_t)dq | (uintptr_t)dk) & 15 || (dq_bs | dq_rs | dq_hs | dk_bs | dk_rs | dk_hs) % unit)
    return mmt_set_error(MMT_EINVAL, "mmt_qk_norm_rope_bwd: rows have to start at multiples of 16 bytes");
  const size_t need = mmt_qk_norm_rope_workspace_bytes(a);
  if (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < need)
    return mmt_set_error(MMT_EINVAL, "mmt_qk_norm_rope_bwd: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, need);
  hipStream_t st = (hipStream_t)stream;
  const Grads g = {dqo, dko, dq_bs, dq_rs, dq_hs, dk_bs, dk_rs, dk_hs, dq, dk, (float *)workspace};
  by_type<true>(a, g, nullptr, nullptr, st);
  const int parts = workgroups(a, true), w_f32 = a->w_dtype == MMT_F32;
  const dim3 grid((2 * a->dh + 15) / 16);
  if (a->dtype == MMT_BF16) hipLaunchKernelGGL(mmt_qk_weight_sum_kernel<__bf16>, grid, dim3(1024), 0, st, g.part, parts, a->dh, w_f32, dq_weight, dk_weight);
  else if (a->dtype == MMT_F16) hipLaunchKernelGGL(mmt_qk_weight_sum_kernel<_Float16>, grid, dim3(1024), 0, st, g.part, parts, a->dh, w_f32, dq_weight, dk_weight);
  else hipLaunchKernelGGL(mmt_qk_weight_sum_kernel<float>, grid, dim3(1024), 0, st, g.part, parts, a->dh, w_f32, dq_weight, dk_weight);
  return status("mmt_qk_norm_rope_bwd");
}
