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
//
// Forms: a sequence of up to 16 rows (queries of one kv head's group) is one 16-column tile and takes
// the short form: 32 single tokens at 4000 keys 47 us, in the long form 111; one at 131071 keys 52 and
// 117.  More rows would be read once per tile of 16; the long form reads 256 (128 above 128 channels) once.
//
// Parts: as many as leave every CU one workgroup.  Up to there each part is so much less work in a
// row; beyond, a second round costs more than it brings (12 tokens at 8000 keys, 96 workgroups: 2
// parts 43 us, 3 parts 61; 40 tokens at 4000, 320 workgroups: whole 81, 2 parts 83, 3 parts 89; 1200
// rows over 4000 keys, 40 tiles: 6 parts 63, 7 parts 83, whole 176).  Parts are joined by a launch of
// 5 us, so short contexts are left whole: a part has at least one step of 64 keys for each wave in the
// short form and a context 3 parts' (one token at 8000 keys 17 us, with 2 steps a wave 20, 4 28; at 1000
// keys 13.0 whole and 12.9 in 2 parts), and 2 steps in the long form and a context 8 (160 rows over 1000
// keys: 2 steps 23.6 us, 4 27.4, 8 36, whole 51; 400 rows over 200 keys: whole 20.3, 2 parts 22.8).
// Beside the long form single tokens wait less for their own work than for CUs: 3 steps a wave
// (a prompt of 200 with two tokens at 8000: 29 us, 1 step 43, 8 steps 64; a prompt of 4000 with four at
// 4000: 247, 248, 240).
Layout layout(const KvAttention &a) {
    Layout l = {};
    const int64_t group = a.q_heads / a.c.kv_heads, t = a.s.num_tokens;
    const int64_t most = a.max_new ? std::min<int64_t>(a.max_new, t) : t;
    l.plan.group = (int)group;
    // where all sequences have more than 16 rows, the long form takes whatever is there
    const bool same = a.max_new && most * a.s.batch == t;
    l.any_long = most * group > attn::SHORT_ROWS;
    l.any_short = group <= attn::SHORT_ROWS && !(same && l.any_long);
    l.plan.short_rows = l.any_short ? attn::SHORT_ROWS : 0;
    // waves of a workgroup, in either form and also all that a CU holds
    const int waves = a.c.head_dim <= 128 ? 8 : 4;
    const int64_t tile_rows = attn::WAVE_ROWS * waves;
    l.plan.tiles = (int)(t * group / tile_rows + a.s.batch);
    const int64_t cus = num_cus(), steps = (a.max_len + attn::TILE - 1) / attn::TILE;
    const auto splits = [&](int64_t wanted, int64_t least, int64_t launched) {
        return (int)std::max<int64_t>(1, std::min({wanted, steps / least, (int64_t)128, MAX_GROUPS / launched}));
    };
    const int64_t sequences = std::min<int64_t>(a.s.batch, t);
    const int64_t groups = sequences * a.c.kv_heads, least = (l.any_long ? 3 : 1) * waves;
    l.plan.splits_short = l.any_short && steps >= 3 * waves ? splits(cus / groups, least, (int64_t)a.s.batch * a.c.kv_heads) : 1;
    // (ragged sequences: the last tile of each is half full in the mean)
    const int64_t tiles = (same ? a.s.batch * ((most * group + tile_rows - 1) / tile_rows) : t * group / tile_rows + (sequences + 1) / 2) * a.c.kv_heads;
    l.plan.splits_long = l.any_long && steps >= 8 ? splits(cus / tiles, 2, (int64_t)l.plan.tiles * a.c.kv_heads) : 1;
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
