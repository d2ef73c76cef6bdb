// Attention with a relative position bias, f16 instances (attn_rel.h).
#include "attn_rel.h"

namespace hk {
template void attn_rel_queue<F16>(const hrt_attn_rel_args&, int, const RelBuckets&, const RelPlan&, hipStream_t);
}  // namespace hk
