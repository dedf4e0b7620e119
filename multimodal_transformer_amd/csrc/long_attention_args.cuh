// What the entry points of attention over long rows (long_attention.hip) hand to the kernels of an element type.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/mmt_amd.h"

namespace la {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4, THREADS = 64 * WAVES, ROWS = 32 * WAVES;   // a workgroup: 4 waves of 32 rows each
constexpr int STAT_PARTS = 256, STAT_THREADS = 1024, STAT_ROWS = STAT_THREADS / 16;   // fp16 maxima: workgroups at most, 16 lanes per row

// Smallest / largest live document id of each tile of keys (or queries); live = id >= 0.
struct DocRange {
  int lo, hi, dead, pad;
};

struct Args {                      // mmt_long_attention plus what the launcher derives
  mmt_long_attention a;
  int G, pack;                     // query heads per key head; heads whose rows share a tile (1 or G)
  int few;                         // all rows of a key head fit into 32: the waves split the keys instead
  int nqt, nkt, nsplit, items;     // row tiles, key tiles, splits of the keys, workgroups
  int teams;                       // forward, dQ: 1, or 2 teams of four waves that deal the key tiles among themselves
  int groups;                      // workgroups n, n + groups, .. share keys and values
  int zh, zq;                      // dK / dV: parts over the query heads of a key head, over the queries
  float *part_dk, *part_dv;        // (zh * zq, B, Lk, Hk, dh) when there are several parts
  const DocRange *krng, *qrng;     // per batch row and tile, or NULL
  void *out, *low;                 // (B, Lq, H, dh); low: what rounding took from out, rounded too, or NULL
  float *lse;                      // (B, H, Lq)
  float *part_o;                   // split: (nsplit, B, H, Lq, dh)
  float *part_ml;                  // split: (nsplit, B, H, Lq, 2): maximum, sum
  // backward
  const void *dout;
  int64_t do_bs, do_rs, do_hs;
  float2 *stat;                    // (B, H, Lq): lse in units of log 2, rowsum(P dP) - dlse
  const f32x4 *maxima;             // fp16: the parts of what bounds the score gradients
  int stat_parts;
  float *dscale;                   // fp16: power of two the score gradients are multiplied by before they are rounded
  void *dq, *dk, *dv;              // (B, Lq, H, dh), (B, Lk, Hk, dh)
  const float *dlse;               // (B, H, Lq) gradient of the log-sum, or NULL
  float *norm;                     // learned bias: (B, H, Lq) 1 / sum of the probabilities as the backward forms them
  float *far_part;                 // (items, 2)
};

template <typename T> void forward(Args &g, DocRange *ranges, hipStream_t st);
template <typename T> void backward(Args &g, DocRange *ranges, f32x4 *maxima, float *table_part, float *dtable, hipStream_t st);

}  // namespace la
