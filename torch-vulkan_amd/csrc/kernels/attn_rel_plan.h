// What the attention kernel with a relative position bias (attn_rel.h) and its launcher (attn_rel.hip) share.
#pragma once

#include "device_common.h"

namespace hk {

// Buckets of one direction: bucket k holds the distances start[k] .. start[k + 1] - 1, the last one all from R = start[nb - 1].
struct RelBuckets {
  int32_t nb, R, sides, total;  // sides 2: positive distances take buckets nb .. 2 nb - 1
  uint16_t start[256];
};

struct RelPlan {
  int g;             // query (key) groups per workgroup
  int nblk;          // workgroups per head along the stationary rows
  int splits, per;   // forward: key ranges and stages in each
};

constexpr int kRelMargin = 63;  // distances of a tile that reaches beyond R on one side

// Streamed rows per stage: a tile per wavefront (two where all four share the keys), fp32 rows of 128 a tile for all.
constexpr int rel_stage(bool f32, int dp, int g) { return f32 && dp > 64 ? 32 : g == 1 ? 128 : 64; }
// Dynamic LDS: the band; for dQ also one band of sums and one 32 x 33 patch per wavefront.
constexpr int rel_lds(int which, int R) { return (2 * R + 1 + 2 * kRelMargin) * 4 * (which == 2 ? 5 : 1) + (which == 2 ? 4 * 32 * 33 * 4 : 0); }

// Queues kernel `which` (0 forward, 1 dK/dV, 2 dQ and the table's partial sums) for element type T.
template <typename T>
void attn_rel_queue(const hrt_attn_rel_args& a, int which, const RelBuckets& bk, const RelPlan& pl, hipStream_t s);

}  // namespace hk
