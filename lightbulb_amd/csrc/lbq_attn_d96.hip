// lbq_attn_d96.hip -- attention over the 8-bit cache (lbq_attn_kernels.hpp), head_dim 96.
#include "lbq_attn_kernels.hpp"

namespace lbq {
hipError_t launch_attn_d96(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st) {
    return attn::launch_dim<96>(a, plan, any_short, any_long, st);
}
}  // namespace lbq
