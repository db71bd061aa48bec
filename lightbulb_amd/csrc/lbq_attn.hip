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
// the short form: 32 single tokens at 4000 keys 45 us, in the long form 111; one at 131071 keys 50 and
// 117.  More rows are more tiles, which read the keys again but out of the caches; the long form reads 256
// rows (128 above 128 channels) once, and has one wave of eight at work for each 32.  Where no sequence has more
// than 48 rows the short form takes all (5 tokens of 4 heads, 32 sequences at 2000 keys: 41 us and 61, 8 at 4000: 25
// and 40; 12 tokens: 57 and 65, 31 and 42), or 64 where their tiles fit the CUs at once (16 tokens, 8
// sequences: 31 and 43; 32, which do not fit: 73 and 65).  Beside longer sequences it takes those of one
// tile (2 tiles: a prompt of 200 with two tokens at 8000 keys 36 us, one tile 31).
//
// Parts: as many as leave every CU one workgroup.  Up to there each part is so much less work in a
// row; beyond, a second filling of the CUs costs more than it brings (12 tokens at 8000 keys, 96 workgroups: 2
// parts 40 us, 3 parts 55; 40 tokens at 4000, 320 workgroups: whole 76, 2 parts 76, 3 parts 80; 1200
// rows over 4000 keys, 40 tiles: 6 parts 60, 7 parts 82, whole 176).  Workgroups of the short form are counted by the
// batch's tokens, not by the most that each sequence could have (12 single tokens at 4000 keys without max_new 26.4
// us, by the most 31; 12 tokens of 6 sequences at 3000, up to 5 each, 18.8 and 22.9).  Parts are joined by a launch of
// 4 to 5 us, so that short contexts are left whole: in the short form up to 2 steps a wave of 64 keys of 128
// channels (1100 keys: whole 13.3 us, parts 11.8 to 12.3; 800: 11.7, 11.8; at 64 channels 1100: 9.5, 11.9), in
// the long form up to 7 steps (400 rows over 200 keys: whole 20.3, 2 parts 22.8).  A part has at
// least 2 steps (short form, 8000 keys of one head: 62 parts 11.9 us, 125 14.1, 31 13.2, 15 14.8; long form, 160 rows
// over 1000 keys: 2 steps 23.6 us, 4 27.4, 8 36, whole 51).  Beside the long form single tokens get
// the CUs that it leaves, and parts of 2 steps a wave (a prompt of 100 with eight tokens at 3000 keys:
// 24 us, 3 steps 30; of 200 with two at 8000: 34, 29, without limit 35); and parts of no more than 16
// steps a wave where it leaves none (a prompt of 4000 with one token at 131071 keys: 279 us,
// 8 steps 300, 32 286, whole 797), but no more than four workgroups a CU: max_len may be far above
// the real lengths (a chunk of 512 with 63 tokens at 2000 keys, max_len 131072: 94 us, without limit 258, two a CU 80; with
// 255 at 1000 keys 160 and 898; with 15 at 2000 and one at 131071 131, 128 and 268).
Layout layout(const KvAttention &a) {
    Layout l = {};
    const int64_t group = a.q_heads / a.c.kv_heads, t = a.s.num_tokens;
    const int64_t most = a.max_new ? std::min<int64_t>(a.max_new, t) : t;
    l.plan.group = (int)group;
    // where all sequences have more rows than the short form takes, the long form takes whatever is there
    const bool same = a.max_new && most * a.s.batch == t;
    const int64_t cus = num_cus(), heads = (int64_t)a.s.batch * a.c.kv_heads;
    const int64_t row_tiles = (most * group + attn::SHORT_ROWS - 1) / attn::SHORT_ROWS, limit = 4 * heads <= cus ? 4 : heads <= MAX_GROUPS / 4 ? 3 : 1;
    const int64_t short_tiles = row_tiles <= limit ? row_tiles : 1;
    const int64_t short_rows = short_tiles * attn::SHORT_ROWS;
    l.any_long = most * group > short_rows;
    l.any_short = group <= short_rows && !(same && l.any_long);
    l.plan.short_rows = l.any_short ? (int)short_rows : 0;
    l.plan.short_tiles = (int)short_tiles;
    // waves of a workgroup, in either form and also all that a CU holds
    const int waves = a.c.head_dim <= 128 ? 8 : 4;
    const int64_t tile_rows = attn::WAVE_ROWS * waves;
    // Workgroups are dealt out to the shader engines in turn, whatever they do: with idle ones between the
    // others some engines have too many (32 sequences of 5 tokens at 2000 keys, 256 tiles and 16 empty ones: 118 and 61).  So tiles are a
    // number for each sequence, where that is no more than by their rows; and where sequences may be idle or
    // of the other form, up to 256 of them are counted by each workgroup for itself (32 tokens, every
    // second of 64 sequences: 60 and 45 us, every fourth of 128: 117 and 45; a few more cycles a workgroup).
    l.plan.listed = a.s.batch > 1 && a.s.batch <= attn::LISTED && !same;
    l.plan.short_groups = (int)((l.plan.listed ? std::min<int64_t>(a.s.batch, t) : a.s.batch) * short_tiles);
    const int64_t per_sequence = (most * group + tile_rows - 1) / tile_rows, by_rows = t * group / tile_rows + a.s.batch;
    l.plan.tiles_per = a.max_new && per_sequence * a.s.batch <= by_rows ? (int)per_sequence : 0;
    l.plan.tiles = (int)(l.plan.tiles_per ? per_sequence * a.s.batch : by_rows);
    // keys that any of a sequence's rows sees
    const int64_t seen = a.causal && a.window > 0 ? std::min<int64_t>(a.max_len, a.window + most) : a.max_len;
    const int64_t steps = (seen + attn::TILE - 1) / attn::TILE;
    const auto splits = [&](int64_t wanted, int64_t least, int64_t launched) {
        return (int)std::max<int64_t>(1, std::min({wanted, steps / least, (int64_t)128, MAX_GROUPS / launched}));
    };
    const int64_t sequences = std::min<int64_t>(a.s.batch, t);
    // (ragged sequences: the last tile of each is half full in the mean)
    const int64_t tiles = (l.plan.tiles_per ? l.plan.tiles : t * group / tile_rows + (sequences + 1) / 2) * a.c.kv_heads;
    l.plan.splits_long = l.any_long && steps >= 8 ? splits(cus / tiles, 2, (int64_t)l.plan.tiles * a.c.kv_heads) : 1;
    // (of the short form: no sequence has fewer than its first token's, and the others' rows fill theirs)
    const int64_t first = (group + attn::SHORT_ROWS - 1) / attn::SHORT_ROWS, more = ((t - sequences) * group + attn::SHORT_ROWS - 1) / attn::SHORT_ROWS;
    const int64_t groups = std::min(sequences * first + more, sequences * short_tiles) * a.c.kv_heads, least = l.any_long ? 2 * waves : 2;
    const int64_t wanted = l.any_long ? std::max((cus - tiles) / groups, std::min(steps / (16 * waves), 4 * cus / groups)) : cus / groups;
    l.plan.splits_short = l.any_short && steps * a.c.head_dim > 256 * waves ? splits(wanted, least, (int64_t)l.plan.short_groups * a.c.kv_heads) : 1;
    const int64_t per = short_rows / group;
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
