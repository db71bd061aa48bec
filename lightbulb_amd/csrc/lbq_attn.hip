// lbq_attn.hip -- attention over the 8-bit paged cache: how a call's work is laid out.
#include "lbq_attn_kernels.hpp"

#include <algorithm>

#include "lbq_internal.hpp"

namespace lbq {
namespace {

struct Layout {
    AttnPlan plan;
    bool any_short, any_long;
    int64_t short_rows, long_rows;  // of one part
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
    const auto splits = [&](int64_t groups, int64_t least, int64_t launched) {
        return (int)std::max<int64_t>(1, std::min({(cus + groups - 1) / groups, steps / least, (int64_t)128, MAX_GROUPS / launched}));
    };
    const int64_t sequences = std::min<int64_t>(a.s.batch, t);
    l.plan.splits_short = l.any_short ? splits(sequences * a.c.kv_heads, (l.any_long ? 8 : 2) * waves, (int64_t)a.s.batch * a.c.kv_heads) : 1;
    // a sequence's last tile is half full in the mean
    const int64_t tiles = (t * group / tile_rows + (sequences + 1) / 2) * a.c.kv_heads;
    l.plan.splits_long = l.any_long && 2 * tiles < cus ? splits(tiles, 4, (int64_t)l.plan.tiles * a.c.kv_heads) : 1;
    const int64_t per = attn::SHORT_ROWS / group;
    l.plan.short_per = l.any_short && per * a.s.batch < t ? (int)per : 0;
    l.plan.short_tokens = l.plan.short_per ? per * a.s.batch : t;
    l.short_rows = l.plan.short_tokens * a.q_heads;
    l.long_rows = t * a.q_heads;
    return l;
}

// rows of parts in the workspace
int64_t part_rows(const Layout &l) {
    return (l.plan.splits_short > 1 ? l.plan.splits_short * l.short_rows : 0) + (l.plan.splits_long > 1 ? l.plan.splits_long * l.long_rows : 0);
}
size_t row_bytes(const KvAttention &a) { return (a.c.head_dim + 2) * sizeof(float); }

}  // namespace

size_t kv_attention_workspace(const KvAttention &a) {
    return a.s.num_tokens ? part_rows(layout(a)) * row_bytes(a) : 0;
}

hipError_t launch_kv_attention(const KvAttention &a, hipStream_t st) {
    Layout l = layout(a);
    // as many parts as there is room for, single tokens' first
    int64_t room = (int64_t)std::min<size_t>(a.ws_bytes / row_bytes(a), INT64_MAX);
    l.plan.splits_short = (int)std::max<int64_t>(1, std::min<int64_t>(l.plan.splits_short, room / l.short_rows));
    if (l.plan.splits_short > 1) room -= l.plan.splits_short * l.short_rows;
    l.plan.splits_long = (int)std::max<int64_t>(1, std::min<int64_t>(l.plan.splits_long, room / l.long_rows));
    l.plan.long_row = l.plan.splits_short > 1 ? l.plan.splits_short * l.short_rows : 0;
    l.plan.part = static_cast<float *>(a.ws);
    l.plan.stat = l.plan.part + part_rows(l) * a.c.head_dim;
    auto launch = a.c.head_dim == 64 ? launch_attn_d64 : a.c.head_dim == 96 ? launch_attn_d96 : a.c.head_dim == 128 ? launch_attn_d128
                  : a.c.head_dim == 192 ? launch_attn_d192 : launch_attn_d256;
    return launch(a, l.plan, l.any_short, l.any_long, st);
}

}  // namespace lbq
