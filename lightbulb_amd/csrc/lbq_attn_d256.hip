// lbq_attn_d256.hip -- attention over the 8-bit cache (lbq_attn_kernels.hpp), head_dim 256.
#include "lbq_attn_kernels.hpp"

namespace lbq {
hipError_t launch_attn_d256(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st) {
    return attn::launch_dim<256>(a, plan, any_short, any_long, st);
}
}  // namespace lbq
