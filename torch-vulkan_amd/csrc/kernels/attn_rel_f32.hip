// Attention with a relative position bias, f32 instances (attn_rel.h).
#include "attn_rel.h"

namespace hk {
template void attn_rel_queue<F32>(const hrt_attn_rel_args&, int, const RelBuckets&, const RelPlan&, hipStream_t);
}  // namespace hk
