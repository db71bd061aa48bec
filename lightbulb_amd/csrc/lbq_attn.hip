// lbq_attn.hip -- attention over the 8-bit paged cache: how a call's work is laid out.
#include "lbq_attn_kernels.hpp"

#include <algorithm>

#include "lbq_internal.hpp"

namespace lbq {
namespace {

struct Layout {
    AttnPlan plan;
    bool any_short, any_long;
    size_t part_bytes;  // per split
};

// Which forms a call needs and into how many parts each cuts a sequence's keys.  The batch's real
// lengths are on the device: the counts go by the bounds that the caller gave.
Layout layout(const KvAttention &a) {
    Layout l = {};
    const int64_t group = a.q_heads / a.c.kv_heads, t = a.s.num_tokens;
    const int64_t most = a.max_new ? std::min<int64_t>(a.max_new, t) : t;
    l.plan.group = (int)group;
    // the short form takes sequences of up to 16 rows, unless all have more (the long form then
    // takes whatever is there)
    const bool same = a.max_new && most * a.s.batch == t;
    l.any_long = most * group > attn::SHORT_ROWS;
    l.any_short = group <= attn::SHORT_ROWS && !(same && l.any_long);
    l.plan.short_rows = l.any_short ? attn::SHORT_ROWS : 0;
    // waves of a workgroup, in either form and also all that a CU holds
    const int waves = a.c.head_dim <= 128 ? 8 : 4;
    const int64_t tile_rows = attn::WAVE_ROWS * waves;
    l.plan.tiles = (int)(t * group / tile_rows + a.s.batch);
    // parts: enough workgroups for every CU, while a part keeps `least` steps of 64 keys
    const int64_t cus = num_cus(), steps = (a.max_len + attn::TILE - 1) / attn::TILE;
    const auto splits = [&](int64_t groups, int64_t least) {
        return (int)std::max<int64_t>(1, std::min({(cus + groups - 1) / groups, steps / least, (int64_t)128}));
    };
    l.plan.splits_short = l.any_short ? splits(std::min<int64_t>(a.s.batch, t) * a.c.kv_heads, (l.any_long ? 8 : 2) * waves) : 1;
    const int64_t tiles = (t * group / tile_rows + 1) * a.c.kv_heads;
    l.plan.splits_long = l.any_long && 2 * tiles < cus ? splits(tiles, 4) : 1;
    l.part_bytes = (size_t)t * a.q_heads * (a.c.head_dim + 2) * sizeof(float);
    return l;
}

}  // namespace

size_t kv_attention_workspace(const KvAttention &a) {
    if (a.s.num_tokens == 0) return 0;
    const Layout l = layout(a);
    const int splits = std::max(l.plan.splits_short, l.plan.splits_long);
    return splits > 1 ? splits * l.part_bytes : 0;
}

hipError_t launch_kv_attention(const KvAttention &a, hipStream_t st) {
    Layout l = layout(a);
    const int room = (int)std::min<size_t>(a.ws_bytes / l.part_bytes, 128);
    l.plan.splits_short = std::max(1, std::min(l.plan.splits_short, room));
    l.plan.splits_long = std::max(1, std::min(l.plan.splits_long, room));
    const int splits = std::max(l.plan.splits_short, l.plan.splits_long);
    l.plan.part = static_cast<float *>(a.ws);
    l.plan.stat = l.plan.part + (size_t)splits * a.num_q * a.q_heads * a.c.head_dim;
    auto launch = a.c.head_dim == 64 ? launch_attn_d64 : a.c.head_dim == 96 ? launch_attn_d96 : a.c.head_dim == 128 ? launch_attn_d128
                  : a.c.head_dim == 192 ? launch_attn_d192 : launch_attn_d256;
    return launch(a, l.plan, l.any_short, l.any_long, st);
}

}  // namespace lbq
