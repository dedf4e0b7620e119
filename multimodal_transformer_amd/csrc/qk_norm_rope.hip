// Norm of queries and keys per head + rotation of their positions in one pass over memory (mmt_qk_norm_rope_fwd / _bwd).
//
// A group of LPH lanes (the power of two at or above dh / 8) holds one head of one token, 8 elements per lane: the mean square and,
// backwards, the dot product are butterflies inside the group, everything else stays in the lane; with the half-split pairing a
// pair's other element comes from the lane rot / 16 further on.  The angles of a token are shared by all its heads: a workgroup
// forms them once per token, in 64 bits (position * frequency reaches 10^6 turns, of which fp32 would keep 2 digits), reduces them to
// a fraction of a turn and keeps cosine and sine in LDS.  Bound by memory: every element is read once and written once (backwards:
// two read, one written).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mmt_amd.h"

int mmt_set_error(int code, const char *fmt, ...);   // transformer.hip

namespace {

constexpr int NT = 256, MAX_PARTS = 1024;

template <typename T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

template <typename T> __device__ __forceinline__ void load8(const T *p, float *x) {
  const typename Vec8<T>::type v = *(const typename Vec8<T>::type *)p;
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

// the pair partners of a lane's 8 elements (half-split pairing): from the lanes that hold them, or element by element when a half is
// no whole number of lanes.  v: this lane's elements; row / w: where to fetch them (value = row[d] * scale(d))
template <int LPH> __device__ __forceinline__ void partners(const float *v, float *o, int lane_in, int half) {
  const int base = (threadIdx.x & 63) - lane_in, step = half / 8;
  const int src = base + ((lane_in < step ? lane_in + step : lane_in - step) & (LPH - 1));
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = __shfl(v[e], src);
}

template <typename T, int LPH, bool BWD> __global__ void __launch_bounds__(NT) mmt_qk_norm_rope_kernel(const mmt_qk_norm_rope a, const Grads g, void *q_out, void *k_out, int tok) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float2 *cs = (float2 *)smem;
  const int lane_in = threadIdx.x % LPH, group = threadIdx.x / LPH, d0 = lane_in * 8, half = a.rot / 2, heads = a.H + a.Hk;
  constexpr int GROUPS = NT / LPH;
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
    __syncthreads();
    angles(a, t0, nt, cs);
    __syncthreads();
    for (int u0 = 0; u0 < nt * heads; u0 += GROUPS) {
      const int u = u0 + group;
      const bool live = u < nt * heads;
      const int lt = live ? u / heads : 0, hh = live ? u % heads : 0;
      const bool is_k = hh >= a.H;
      const int hd = is_k ? hh - a.H : hh;
      const int64_t t = t0 + lt, b = t / a.L, i = t % a.L;
      const T *row = is_k ? (const T *)a.k + b * a.k_bs + i * a.k_rs + hd * a.k_hs : (const T *)a.q + b * a.q_bs + i * a.q_rs + hd * a.q_hs;
      const int64_t oi = is_k ? (t * a.Hk + hd) * a.dh : (t * a.H + hd) * a.dh;
      const void *wrow = is_k ? a.k_weight : a.q_weight;
      float x[8] = {}, gy[8] = {};
      if (live && on) load8(row + d0, x);
      const T *grow = nullptr;
      if (BWD) {
        grow = is_k ? (const T *)g.dko + b * g.k_bs + i * g.k_rs + hd * g.k_hs : (const T *)g.dqo + b * g.q_bs + i * g.q_rs + hd * g.q_hs;
        if (live && on) load8(grow + d0, gy);
      }
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
      for (int m = 1; m < LPH; m <<= 1) ss += __shfl_xor(ss, m);
      const float r = 1.f / sqrtf(ss / (float)a.dh + a.eps);
      float v[8], o[8];                       // what is turned (forward: the norm, backward: the gradient), and its partners
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = BWD ? gy[e] : x[e] * r * (is_k ? wk[e] : wq[e]);
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e ^ 1];
      } else if (by_lane) {
        partners<LPH>(v, o, lane_in, half);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = d0 + e, p = d < half ? d + half : d - half;
          o[e] = 0.f;
          if (live && on && d < a.rot)
            o[e] = BWD ? (float)grow[p] : (float)row[p] * r * weight_at<T>(wrow, a.w_dtype == MMT_F32, p);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        if (d < a.rot) {
          const bool first = a.interleaved ? !(d & 1) : d < half;
          const float2 c = cs[lt * half + (a.interleaved ? d >> 1 : first ? d : d - half)];
          const float s = first != BWD ? -c.y : c.y;         // forward: (-, +) for (first, second); the gradient turns back
          v[e] = fmaf(o[e], s, v[e] * c.x);
        }
      }
      if (!BWD) {
        if (live && on) store8((T *)(is_k ? k_out : q_out) + oi + d0, v);
      } else {
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float c = live ? v[e] * x[e] * r : 0.f;
          if (is_k) sk[e] += c;
          else sq[e] += c;
          v[e] *= is_k ? wk[e] : wq[e];
          dot = fmaf(v[e], x[e], dot);
        }
#pragma unroll
        for (int m = 1; m < LPH; m <<= 1) dot += __shfl_xor(dot, m);
        const float f = dot * r * r / (float)a.dh;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r * fmaf(-f, x[e], v[e]);
        if (live && on) store8((T *)(is_k ? g.dk : g.dq) + oi + d0, v);
      }
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

// parts -> weight gradients, in 64 bits and in a fixed order: 16 threads per element
template <typename T> __global__ void mmt_qk_weight_sum_kernel(const float *part, int parts, int dh, int w_f32, void *dqw, void *dkw) {
  const int n = blockIdx.x * 16 + (threadIdx.x >> 4), s = threadIdx.x & 15;
  const bool on = n < 2 * dh;
  double v = 0.;
  if (on)
    for (int p = s; p < parts; p += 16) v += part[(int64_t)p * 2 * dh + n];
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) v += __shfl_xor(v, m);
  if (!on || s) return;
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

// tokens per workgroup and step: several share the angles' latency, but few tokens are spread over the chip
int tokens_per_group(const mmt_qk_norm_rope *a) { return (int64_t)a->B * a->L < 4096 ? 1 : 4; }
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
  hipLaunchKernelGGL((mmt_qk_norm_rope_kernel<T, LPH, BWD>), dim3(workgroups(a, BWD)), dim3(NT), lds, st, *a, g, qo, ko, tok);
}
template <typename T, bool BWD> void by_size(const mmt_qk_norm_rope *a, const Grads &g, void *qo, void *ko, hipStream_t st) {
  if (a->dh <= 32) go<T, 4, BWD>(a, g, qo, ko, st);
  else if (a->dh <= 64) go<T, 8, BWD>(a, g, qo, ko, st);
  else if (a->dh <= 128) go<T, 16, BWD>(a, g, qo, ko, st);
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
  if (a->dtype == MMT_BF16) hipLaunchKernelGGL(mmt_qk_weight_sum_kernel<__bf16>, grid, dim3(256), 0, st, g.part, parts, a->dh, w_f32, dq_weight, dk_weight);
  else if (a->dtype == MMT_F16) hipLaunchKernelGGL(mmt_qk_weight_sum_kernel<_Float16>, grid, dim3(256), 0, st, g.part, parts, a->dh, w_f32, dq_weight, dk_weight);
  else hipLaunchKernelGGL(mmt_qk_weight_sum_kernel<float>, grid, dim3(256), 0, st, g.part, parts, a->dh, w_f32, dq_weight, dk_weight);
  return status("mmt_qk_norm_rope_bwd");
}
