// Attention over long rows (no counterpart in the reference, whose longest row is a few dozen tokens: mgcvae.py:276-282,375-449):
//   mmt_long_attention_fwd / _bwd   capped scores, distance bias, learned bucket bias, document / prefix / causal masks, cache
//                                   lengths, shared key heads; bf16, fp16, fp32; forward, backward, few rows over a long cache
// The kernels are in long_attention_kernels.cuh; mmt_attention_fwd / _bwd (train.hip) stay the path for rows of at most 32 keys with
// stored probabilities.
#include <algorithm>

#include "long_attention_args.cuh"

int mmt_set_error(int code, const char *fmt, ...);   // transformer.hip

namespace la {

static int elem_size(int dtype) { return dtype == MMT_F32 ? 4 : 2; }
static int tile_keys(int dtype) { return dtype == MMT_F32 ? 32 : 64; }

static int check(const mmt_long_attention *a, const char *who) {
  if (!a || !a->q || !a->k || !a->v) return mmt_set_error(MMT_EINVAL, "%s: null pointer", who);
  if (a->dtype != MMT_F32 && a->dtype != MMT_BF16 && a->dtype != MMT_F16)
    return mmt_set_error(MMT_EINVAL, "%s: unknown element type %d", who, a->dtype);
  if (a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->Lq <= 0 || a->Lk <= 0)
    return mmt_set_error(MMT_EINVAL, "%s: B, H, Hk, Lq and Lk have to be positive", who);
  if (a->H % a->Hk) return mmt_set_error(MMT_EINVAL, "%s: %d query heads are no multiple of %d key heads", who, a->H, a->Hk);
  if (a->dh < 8 || a->dh > 128 || a->dh % 8) return mmt_set_error(MMT_EINVAL, "%s: head size %d, need a multiple of 8 up to 128", who, a->dh);
  // (also in units of log 2, and divided by one another)
  if (!(a->scale > 0.f) || !isfinite(2.f * a->scale)) return mmt_set_error(MMT_EINVAL, "%s: the scale has to be positive and finite", who);
  if (!(a->softcap >= 0.f) || !isfinite(2.f * a->softcap) || (a->softcap > 0.f && !isfinite(a->scale / a->softcap)))
    return mmt_set_error(MMT_EINVAL, "%s: the cap has to be finite, not negative and not far below the scale", who);
  if (a->prefix && !a->causal) return mmt_set_error(MMT_EINVAL, "%s: a prefix is an exception from the causal mask", who);
  if (!a->q_doc != !a->k_doc) return mmt_set_error(MMT_EINVAL, "%s: documents need ids for the queries and the keys", who);
  if (!a->rel_bias != !a->rel_buckets) return mmt_set_error(MMT_EINVAL, "%s: a learned bias needs its table and its buckets", who);
  if (a->rel_bias && (a->n_buckets < 1 || a->n_buckets > 64 || a->reach < 1 || a->reach > 1024))
    return mmt_set_error(MMT_EINVAL, "%s: need 1..64 buckets and a reach of 1..1024", who);
  if (a->Lk > (1 << 30) || a->Lq > (1 << 30)) return mmt_set_error(MMT_EINVAL, "%s: at most 2^30 tokens per row", who);
  const int64_t unit = 16 / elem_size(a->dtype);
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) & 15 ||
      (a->q_bs | a->q_rs | a->q_hs | a->k_bs | a->k_rs | a->k_hs | a->v_bs | a->v_rs | a->v_hs) % unit)
    return mmt_set_error(MMT_EINVAL, "%s: rows of q, k and v have to start at multiples of 16 bytes", who);
  const int64_t far = ((int64_t)1 << 31) / 64 / elem_size(a->dtype);       // 64 rows are addressed with 32 bits
  if (a->q_rs >= far || a->k_rs >= far || a->v_rs >= far || a->q_rs < 0 || a->k_rs < 0 || a->v_rs < 0)
    return mmt_set_error(MMT_EINVAL, "%s: token strides have to stay below 2^25 bytes", who);
  // (a launch has fewer than 2^32 threads, 512 to a workgroup)
  const double items = (double)a->B * a->H * (((double)a->Lq + ROWS - 1) / ROWS) + (double)a->B * a->Hk * (((double)a->Lk + ROWS - 1) / ROWS);
  const double sums = a->rel_bias ? 64. * a->H * a->n_buckets : 0.;                 // one wave for each entry of the table
  if (items > 8e6 || (double)a->B * a->H * a->Lq > 2e9 || sums >= 4294967296.) return mmt_set_error(MMT_EINVAL, "%s: too many rows for one call", who);
  return MMT_OK;
}

// One workgroup of 128 rows per CU leaves each SIMD one wave, which waits for most of its time: two teams of waves then share its keys.
// Where that many rows are causal, the workgroups that remain for a second turn are the shortest.  Measured with one team and two: bf16
// causal 2 x 1024 x 16 heads of 64 (256 workgroups) forward 23 and 21 us, dQ 27 and 24; fp16 causal 3 x 1333 x 8 heads of 80 (264) with a
// learned bias 47 and 37, 63 and 50.  fp32 needs the registers of both.
static int teams(const mmt_long_attention &a, int64_t items) {
  return a.dtype != MMT_F32 && items < (a.causal ? 512 : 257) && a.Lk > 192 ? 2 : 1;
}

static void plan(Args &g, bool backward) {
  const mmt_long_attention &a = g.a;
  const int bk = tile_keys(a.dtype);
  g.G = a.H / a.Hk;
  // few queries: the rows of all heads that share a key head go into one tile of 32, which reads the cache once (32768 tokens, one query
  // of 4 heads per key head: 285 us instead of 914)
  g.few = !backward && (int64_t)a.Lq * g.G <= 32;
  // else packed where rows of one head would leave more of the tiles of 128 empty (64 queries of 4 heads over 16384 tokens: 38 us instead
  // of 56); a learned bias is laid out for one head
  const bool fewer = ((int64_t)a.Lq * g.G + ROWS - 1) / ROWS < (int64_t)g.G * ((a.Lq + ROWS - 1) / ROWS);
  g.pack = g.few || (!backward && !a.rel_bias && fewer) ? g.G : 1;
  g.nqt = (int)(((int64_t)a.Lq * g.pack + ROWS - 1) / ROWS);
  g.nkt = (a.Lk + bk - 1) / bk;
  g.groups = a.B * a.Hk;
  g.nsplit = g.zh = g.zq = 1;
  if (!backward) {
    const int64_t base = (int64_t)g.groups * (g.G / g.pack) * g.nqt;
    const int64_t tiles = g.few ? (a.Lk + 127) / 128 : g.nkt;               // a step of all waves
    g.teams = g.few ? 1 : teams(a, base);
    // the keys are split where that leaves half of the CUs' places empty, two workgroups of four waves per CU or one of two teams: 37 + 10 us
    // with the joining kernel for the chunk above with one team, 38 + 7 with two, with half as many workgroups 57 + 5; at least four tiles to a
    // team, and no split above half (264 workgroups of one team split in two: 32 + 18 us, whole 46)
    const int64_t want = 512 / g.teams;
    if (base < want / 2) g.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>((want + base - 1) / base, tiles / (4 * g.teams)));
    g.items = (int)(base * g.nsplit);
  } else {
    // parts of dK / dV over the query heads, then over the queries, for 512 workgroups, for causal rows, which are uneven, 1024 (bf16 8192 x
    // 16 heads of 128 over 4: 618 us and 23 for the sum of the parts, for 512 609 and 14, for 256 1113; packed scenes of 2 x 4096 tokens 79 and
    // 13, for 512 99 and 8, for 256 187); at least eight tiles of queries each (fp16 3 x 1333 x 8 heads of 80 over 2: 48 and 8 us, with four 64
    // and 13).  All of these were chosen on 16-bit types; fp32 takes them as they are.
    const int64_t base = (int64_t)g.groups * ((a.Lk + ROWS - 1) / ROWS), want = ((a.causal ? 1024 : 512) + base - 1) / base;
    g.zh = (int)std::min<int64_t>(g.G, want);
    g.teams = teams(a, (int64_t)a.B * a.H * g.nqt);
    g.zq = (int)std::max<int64_t>(1, std::min<int64_t>(want / g.zh, (a.Lq + bk - 1) / bk / 8));
  }
}

static size_t align64(size_t n) { return (n + 63) & ~(size_t)63; }

struct Workspace {                 // one piece after another, each a multiple of 64 bytes
  size_t docs, part_o, part_ml, stat, maxima, norm, far, table, part_dk, part_dv, total;
};
static Workspace layout(const Args &g, bool backward) {
  const mmt_long_attention &a = g.a;
  Workspace w = {};
  const size_t rows = (size_t)a.B * a.H * a.Lq, bk = tile_keys(a.dtype);
  size_t n = 0;
  if (a.q_doc) w.docs = n, n += align64(sizeof(DocRange) * a.B * ((a.Lk + bk - 1) / bk + (a.Lq + bk - 1) / bk));
  if (!backward) {
    if (g.nsplit > 1) {
      w.part_o = n, n += align64(4 * rows * a.dh * g.nsplit);
      w.part_ml = n, n += align64(8 * rows * g.nsplit);
    }
  } else {
    w.stat = n, n += align64(8 * rows);
    if (a.dtype == MMT_F16) w.maxima = n, n += 16 * (STAT_PARTS + 4);
    if (a.rel_bias) {
      const size_t tiles = (size_t)a.B * g.nqt * a.H;
      w.norm = n, n += align64(4 * rows);
      w.far = n, n += align64(8 * tiles);
      w.table = n, n += align64(4 * tiles * a.n_buckets);
    }
    if (g.zh * g.zq > 1) {
      const size_t part = align64((size_t)4 * g.zh * g.zq * a.B * a.Lk * a.Hk * a.dh);
      w.part_dk = n, n += part;
      w.part_dv = n, n += part;
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
  plan(g, backward != 0);
  return layout(g, backward != 0).total;
}

extern "C" int mmt_long_attention_fwd(const mmt_long_attention *a, void *out, void *out_low, float *lse, void *workspace,
                                      size_t workspace_bytes, void *stream) {
  if (int rc = check(a, "mmt_long_attention_fwd")) return rc;
  if (!out || ((uintptr_t)out | (uintptr_t)out_low) & 15)
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_fwd: out has to be a 16-byte aligned address");
  Args g = {};
  g.a = *a;
  plan(g, false);
  const Workspace w = layout(g, false);
  if (w.total && (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < w.total))
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_fwd: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, w.total);
  char *ws = (char *)workspace;
  g.out = out, g.low = out_low, g.lse = lse;
  g.part_o = (float *)(ws + w.part_o), g.part_ml = (float *)(ws + w.part_ml);
  DocRange *ranges = a->q_doc ? (DocRange *)(ws + w.docs) : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == MMT_BF16) forward<__bf16>(g, ranges, st);
  else if (a->dtype == MMT_F16) forward<_Float16>(g, ranges, st);
  else forward<float>(g, ranges, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MMT_OK : mmt_set_error(MMT_ELAUNCH, "mmt_long_attention_fwd: %s", hipGetErrorString(e));
}

extern "C" int mmt_long_attention_bwd(const mmt_long_attention *a, const void *out, const void *out_low, const float *lse, const void *dout,
                                      int64_t do_bs, int64_t do_rs, int64_t do_hs, const float *dlse, void *dq, void *dk, void *dv,
                                      float *drel_bias, void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = check(a, "mmt_long_attention_bwd")) return rc;
  if (!out || !lse || !dout || !dq || !dk || !dv || (a->rel_bias && !drel_bias))
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_bwd: null pointer");
  if (((uintptr_t)out | (uintptr_t)out_low | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15 ||
      (do_bs | do_rs | do_hs) % (16 / elem_size(a->dtype)) || do_rs < 0 || do_rs >= ((int64_t)1 << 31) / 64 / elem_size(a->dtype))
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_bwd: rows have to start at multiples of 16 bytes, token strides to stay below 2^25 bytes");
  Args g = {};
  g.a = *a;
  plan(g, true);
  const Workspace w = layout(g, true);
  if (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < w.total)
    return mmt_set_error(MMT_EINVAL, "mmt_long_attention_bwd: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, w.total);
  char *ws = (char *)workspace;
  g.out = const_cast<void *>(out), g.low = const_cast<void *>(out_low), g.lse = const_cast<float *>(lse);
  g.dout = dout, g.do_bs = do_bs, g.do_rs = do_rs, g.do_hs = do_hs;
  g.dq = dq, g.dk = dk, g.dv = dv, g.dlse = dlse;
  g.stat = (float2 *)(ws + w.stat);
  if (a->rel_bias) g.norm = (float *)(ws + w.norm), g.far_part = (float *)(ws + w.far);
  if (g.zh * g.zq > 1) g.part_dk = (float *)(ws + w.part_dk), g.part_dv = (float *)(ws + w.part_dv);
  DocRange *ranges = a->q_doc ? (DocRange *)(ws + w.docs) : nullptr;
  float *table = a->rel_bias ? (float *)(ws + w.table) : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == MMT_BF16) backward<__bf16>(g, ranges, nullptr, table, drel_bias, st);
  else if (a->dtype == MMT_F16) backward<_Float16>(g, ranges, (f32x4 *)(ws + w.maxima), table, drel_bias, st);
  else backward<float>(g, ranges, nullptr, table, drel_bias, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MMT_OK : mmt_set_error(MMT_ELAUNCH, "mmt_long_attention_bwd: %s", hipGetErrorString(e));
}
