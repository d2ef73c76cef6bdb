// What the attention kernel with a relative position bias (attn_rel.h) and its launcher (attn_rel.hip) share.
#pragma once

#include "device_common.h"

namespace hk {

// Buckets of one direction: bucket k holds the distances start[k] .. start[k + 1] - 1, the last one all from R = start[nb - 1];
// from start[nb] on: INT32_MAX.
struct RelBuckets {
  int32_t nb, R, sides, total;  // sides 2: positive distances take buckets nb .. 2 nb - 1
  int32_t start[256];
};

struct RelPlan {
  int g;             // query (key) groups per workgroup; 0: forward of one query at a time (attn_rel.hip)
  int nblk;          // workgroups per head along the stationary rows
  int splits, per;   // forward: key ranges and stages in each
  int table;         // dK/dV: workgroups ahead of the others that finish the table's gradient
  int64_t parts;     // partial sums of it per head
};

// The bucket of distance n: how many borders it reaches.  They are scalars, sixteen to a load (one by one, a head's band of
// distances took two microseconds of waits).
__device__ __forceinline__ int rel_bucket(const RelBuckets& bk, int n) {
  int k = -1;
  for (int i = 0; i < bk.nb; i += 16)
#pragma unroll
    for (int j = 0; j < 16; ++j) k += n >= bk.start[i + j];
  return k;
}

constexpr int kRelMargin = 63;  // distances of a tile that reaches beyond R on one side

// Streamed rows per stage: a tile per wavefront (two where all four share the keys), fp32 rows of 128 a tile for all.
constexpr int rel_stage(bool f32, int dp, int g) { return f32 && dp > 64 ? 32 : g == 1 ? 128 : 64; }
// Dynamic LDS: the band; for dQ also one band of sums and one 32 x 33 patch per wavefront.
constexpr int rel_lds(int which, int R) { return (2 * R + 1 + 2 * kRelMargin) * 4 * (which == 2 ? 5 : 1) + (which == 2 ? 4 * 32 * 33 * 4 : 0); }

// dtable[k, h] = the workgroups' partial sums [H][n][buckets], value i by one wavefront: lanes stride the partial sums, then
// one fixed exchange.
template <typename T>
__device__ __forceinline__ void rel_table(const hrt_attn_rel_args& p, int64_t n, int64_t i, int lane) {
  if (i >= (int64_t)p.buckets * p.H) return;
  const int64_t h = i / p.buckets, k = i % p.buckets;
  const HK_G float* part = gcptr<float>(p.ws) + h * n * p.buckets + k;
  float s = 0.f;
  for (int64_t j = lane; j < n; j += 64) s += part[j * p.buckets];
  s = wave_sum(s);
  if (lane == 0) gptr<typename T::storage>(p.dtable)[k * p.H + h] = T::from_f32(s);
}

// Queues kernel `which` (0 forward, 1 dK/dV, 2 dQ and the table's partial sums) for element type T.
template <typename T>
void attn_rel_queue(const hrt_attn_rel_args& a, int which, const RelBuckets& bk, const RelPlan& pl, hipStream_t s);

}  // namespace hk
