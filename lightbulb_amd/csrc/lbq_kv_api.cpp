// lbq_kv_api.cpp -- C entry points of the 8-bit paged key/value cache (include/lbq.h): the
// arguments' checks and the launches.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>

#include "../../include/lbq.h"
#include "lbq_kv.hpp"

// lbq_api.cpp
int lbq_fail_status(int status, const char *msg);
int lbq_ctx_device(const lbq_ctx *ctx);

namespace {

int fail(int status, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return lbq_fail_status(status, buf);
}

// the context's device for the length of a call
struct OnDevice {
    int prev = -1, dev;
    hipError_t err = hipSuccess;
    explicit OnDevice(const lbq_ctx *ctx) : dev(lbq_ctx_device(ctx)) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != dev) err = hipSetDevice(dev);
    }
    ~OnDevice() {
        if (prev >= 0 && prev != dev) (void)hipSetDevice(prev);
    }
};

template <class Launch>
int launched(const lbq_ctx *ctx, const char *what, Launch launch) {
    OnDevice on(ctx);
    hipError_t e = on.err != hipSuccess ? on.err : launch();
    return e == hipSuccess ? LBQ_OK : fail(LBQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool aligned(const void *p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int MAX_BATCH = 65536;
constexpr int64_t MAX_TOKENS = (int64_t)1 << 24;
constexpr int MAX_HEADS = 1024;
constexpr int64_t MAX_LEN = (int64_t)1 << 30;

int log2_of_page(int page_size) {
    return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : -1;
}

int check_page(int32_t page_size) {
    if (log2_of_page(page_size) < 0) return fail(LBQ_ERR_SHAPE, "page size %d is none of 16, 32, 64 and 128", page_size);
    return LBQ_OK;
}

int check_tables(const int32_t *tables, int64_t stride, int32_t max_blocks, int32_t batch) {
    if (!tables) return fail(LBQ_ERR_INVALID_ARG, "null block tables");
    if (!aligned(tables, 4)) return fail(LBQ_ERR_INVALID_ARG, "block tables must be 4-byte aligned");
    if (batch < 1) return fail(LBQ_ERR_SHAPE, "a batch of %d sequences", batch);
    if (batch > MAX_BATCH) return fail(LBQ_ERR_LIMIT, "a batch of %d sequences exceeds %d", batch, MAX_BATCH);
    if (max_blocks < 1 || stride < max_blocks)
        return fail(LBQ_ERR_SHAPE, "%d blocks in table rows of %lld", max_blocks, (long long)stride);
    return LBQ_OK;
}

int check_cache(const lbq_kv_cache *c, lbq::KvCacheView *v) {
    if (!c) return fail(LBQ_ERR_INVALID_ARG, "null cache");
    if (!c->d_k || !c->d_v || !c->d_k_scales || !c->d_v_scales) return fail(LBQ_ERR_INVALID_ARG, "null codes or scales in the cache");
    if (!aligned(c->d_k, 16) || !aligned(c->d_v, 16)) return fail(LBQ_ERR_INVALID_ARG, "the cache's codes must be 16-byte aligned");
    if (!aligned(c->d_k_scales, 4) || !aligned(c->d_v_scales, 4))
        return fail(LBQ_ERR_INVALID_ARG, "the cache's scales must be 4-byte aligned");
    if (c->kind != LBQ_KV_INT8 && c->kind != LBQ_KV_E4M3)
        return fail(LBQ_ERR_UNSUPPORTED_TYPE, "cache kind %d is neither int8 (0) nor e4m3 (1)", c->kind);
    if (int s = check_page(c->page_size)) return s;
    const int d = c->head_dim;
    if (d != 64 && d != 96 && d != 128 && d != 192 && d != 256)
        return fail(LBQ_ERR_SHAPE, "head_dim %d is none of 64, 96, 128, 192 and 256", d);
    if (c->kv_heads < 1 || c->num_pages < 1)
        return fail(LBQ_ERR_SHAPE, "a cache of %lld pages and %d heads", (long long)c->num_pages, c->kv_heads);
    if (c->kv_heads > MAX_HEADS || c->num_pages > INT32_MAX)
        return fail(LBQ_ERR_LIMIT, "a cache of %lld pages and %d heads exceeds the supported maximum", (long long)c->num_pages, c->kv_heads);
    *v = {static_cast<uint8_t *>(c->d_k), static_cast<uint8_t *>(c->d_v), c->d_k_scales, c->d_v_scales, c->num_pages, c->kind,
          c->page_size, log2_of_page(c->page_size), c->kv_heads, d};
    return LBQ_OK;
}

int check_step(const lbq_kv_step *s, bool maps, lbq::KvStepView *v) {
    if (!s) return fail(LBQ_ERR_INVALID_ARG, "null step");
    if (int e = check_tables(s->d_tables, s->table_stride, s->max_blocks, s->batch)) return e;
    if (!s->d_seq_lens || !s->d_cu_new || (maps && (!s->d_slots || !s->d_positions)))
        return fail(LBQ_ERR_INVALID_ARG, "null lengths, rows, slots or positions in the step");
    if (!aligned(s->d_seq_lens, 4) || !aligned(s->d_cu_new, 4) || !aligned(s->d_slots, 8) || !aligned(s->d_positions, 4))
        return fail(LBQ_ERR_INVALID_ARG, "the step's arrays must be aligned to their elements");
    if (s->num_tokens < 0 || s->max_len < 0 || s->max_new < 0) return fail(LBQ_ERR_SHAPE, "a negative size in the step");
    if (s->num_tokens > MAX_TOKENS) return fail(LBQ_ERR_LIMIT, "%lld tokens exceed the supported maximum", (long long)s->num_tokens);
    *v = {s->d_tables, s->table_stride, s->d_seq_lens, s->d_cu_new, s->d_slots, s->d_positions, s->num_tokens, s->max_blocks, s->batch};
    return LBQ_OK;
}

int check_dtype(uint32_t t, int *dt) {
    *dt = t == LBQ_TYPE_F32 ? lbq::DT_F32 : t == LBQ_TYPE_F16 ? lbq::DT_F16 : lbq::DT_BF16;
    if (t != LBQ_TYPE_F32 && t != LBQ_TYPE_F16 && t != LBQ_TYPE_BF16)
        return fail(LBQ_ERR_UNSUPPORTED_TYPE, "type %u of q, k and v is none of F32, F16 and BF16", t);
    return LBQ_OK;
}

int check_rows(const char *what, const void *p, int64_t ts, int64_t hs, int dt) {
    if (!p) return fail(LBQ_ERR_INVALID_ARG, "null %s", what);
    if (!aligned(p, dt == lbq::DT_F32 ? 4 : 2)) return fail(LBQ_ERR_INVALID_ARG, "%s must be aligned to its elements", what);
    if (ts < 0 || hs < 0) return fail(LBQ_ERR_SHAPE, "negative strides of %s", what);
    return LBQ_OK;
}

// whether rows [tokens][heads][dim] and a contiguous output share memory
bool overlaps(const void *p, int64_t ts, int64_t hs, int64_t tokens, int heads, int dim, int size, const void *out, int out_heads) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), o = reinterpret_cast<uintptr_t>(out);
    const uintptr_t an = ((uintptr_t)(tokens - 1) * ts + (uintptr_t)(heads - 1) * hs + dim) * size;
    return a < o + (uintptr_t)tokens * out_heads * dim * size && o < a + an;
}

int check_query_heads(int32_t q_heads, int32_t kv_heads) {
    if (q_heads < 1 || q_heads % kv_heads) return fail(LBQ_ERR_SHAPE, "%d query heads over %d key/value heads", q_heads, kv_heads);
    if (q_heads > MAX_HEADS) return fail(LBQ_ERR_LIMIT, "%d query heads exceed %d", q_heads, MAX_HEADS);
    return LBQ_OK;
}

}  // namespace

extern "C" {

int lbq_kv_step_build(lbq_ctx *ctx, const int32_t *d_ctx_lens, const int32_t *d_new_lens, int32_t batch, int32_t *d_tables,
                      int64_t table_stride, int32_t max_blocks, int32_t page_size, const int32_t *d_free, int64_t num_pages,
                      const int32_t *d_free_count, int32_t *d_free_count_out, uint32_t *d_ticket, int64_t num_tokens,
                      int32_t *d_seq_lens, int32_t *d_cu_new, int32_t *d_granted, int64_t *d_slots, int32_t *d_positions,
                      void *stream) {
    if (!ctx || !d_ctx_lens || !d_new_lens || !d_free || !d_free_count || !d_free_count_out || !d_seq_lens || !d_cu_new ||
        !d_granted || (num_tokens > 0 && (!d_slots || !d_positions)))
        return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_kv_step_build");
    if (d_free_count == d_free_count_out && !d_ticket)
        return fail(LBQ_ERR_INVALID_ARG, "a free count updated in place needs a ticket word");
    for (const void *p : {(const void *)d_ctx_lens, (const void *)d_new_lens, (const void *)d_free, (const void *)d_free_count,
                          (const void *)d_free_count_out, (const void *)d_ticket, (const void *)d_seq_lens, (const void *)d_cu_new,
                          (const void *)d_granted, (const void *)d_positions})
        if (!aligned(p, 4)) return fail(LBQ_ERR_INVALID_ARG, "lbq_kv_step_build's arrays must be aligned to their elements");
    if (!aligned(d_slots, 8)) return fail(LBQ_ERR_INVALID_ARG, "slots must be 8-byte aligned");
    if (int e = check_tables(d_tables, table_stride, max_blocks, batch)) return e;
    if (int e = check_page(page_size)) return e;
    if (num_pages < 1 || num_tokens < 0) return fail(LBQ_ERR_SHAPE, "%lld pages, %lld tokens", (long long)num_pages, (long long)num_tokens);
    if (num_pages > INT32_MAX || num_tokens > MAX_TOKENS)
        return fail(LBQ_ERR_LIMIT, "%lld pages or %lld tokens exceed the supported maximum", (long long)num_pages, (long long)num_tokens);
    lbq::KvStepBuild a = {d_ctx_lens, d_new_lens, d_tables, table_stride, d_free, num_pages, d_free_count, d_free_count_out, d_ticket,
                          d_seq_lens, d_cu_new, d_granted, d_slots, d_positions, num_tokens, batch, max_blocks, log2_of_page(page_size)};
    return launched(ctx, "step launch", [&] { return lbq::launch_kv_step(a, static_cast<hipStream_t>(stream)); });
}

int lbq_kv_release(lbq_ctx *ctx, const int32_t *d_lens, const int32_t *d_which, int32_t batch, int32_t *d_tables,
                   int64_t table_stride, int32_t max_blocks, int32_t page_size, int32_t *d_free, int64_t num_pages,
                   int32_t *d_free_count, void *stream) {
    if (!ctx || !d_lens || !d_which || !d_free || !d_free_count) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_kv_release");
    for (const void *p : {(const void *)d_lens, (const void *)d_which, (const void *)d_free, (const void *)d_free_count})
        if (!aligned(p, 4)) return fail(LBQ_ERR_INVALID_ARG, "lbq_kv_release's arrays must be 4-byte aligned");
    if (int e = check_tables(d_tables, table_stride, max_blocks, batch)) return e;
    if (int e = check_page(page_size)) return e;
    if (num_pages < 1) return fail(LBQ_ERR_SHAPE, "%lld pages", (long long)num_pages);
    if (num_pages > INT32_MAX) return fail(LBQ_ERR_LIMIT, "%lld pages exceed the supported maximum", (long long)num_pages);
    lbq::KvRelease a = {d_tables, table_stride, d_lens, d_which, d_free, num_pages, d_free_count, batch, max_blocks, log2_of_page(page_size)};
    return launched(ctx, "release launch", [&] { return lbq::launch_kv_release(a, static_cast<hipStream_t>(stream)); });
}

int lbq_kv_append(lbq_ctx *ctx, const lbq_kv_cache *cache, const lbq_kv_step *step, uint32_t dtype, const void *d_k,
                  int64_t k_token_stride, int64_t k_head_stride, const void *d_v, int64_t v_token_stride, int64_t v_head_stride,
                  const void *d_q, int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads, const float *d_cos,
                  const float *d_sin, int64_t max_pos, int32_t rot_dim, int32_t interleaved, void *d_q_out, void *stream) {
    if (!ctx) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_kv_append");
    lbq::KvAppend a = {};
    if (int e = check_cache(cache, &a.c)) return e;
    if (int e = check_step(step, step && step->num_tokens > 0, &a.s)) return e;
    if (int e = check_dtype(dtype, &a.dtype)) return e;
    if (rot_dim < 0 || rot_dim > a.c.head_dim || rot_dim % 2)
        return fail(LBQ_ERR_SHAPE, "%d rotated channels of %d", rot_dim, a.c.head_dim);
    if (rot_dim && (!d_cos || !d_sin)) return fail(LBQ_ERR_INVALID_ARG, "null angles");
    if (rot_dim && (!aligned(d_cos, 4) || !aligned(d_sin, 4))) return fail(LBQ_ERR_INVALID_ARG, "angles must be 4-byte aligned");
    if (rot_dim && max_pos < 1) return fail(LBQ_ERR_SHAPE, "angles of %lld positions", (long long)max_pos);
    if (a.s.num_tokens == 0) return LBQ_OK;
    if (int e = check_rows("k", d_k, k_token_stride, k_head_stride, a.dtype)) return e;
    if (int e = check_rows("v", d_v, v_token_stride, v_head_stride, a.dtype)) return e;
    if (d_q) {
        if (int e = check_rows("q", d_q, q_token_stride, q_head_stride, a.dtype)) return e;
        if (int e = check_rows("the rotated q", d_q_out, 0, 0, a.dtype)) return e;
        if (q_heads < 1) return fail(LBQ_ERR_SHAPE, "%d query heads", q_heads);
        if (q_heads > MAX_HEADS) return fail(LBQ_ERR_LIMIT, "%d query heads exceed %d", q_heads, MAX_HEADS);
        const int size = a.dtype == lbq::DT_F32 ? 4 : 2, d = a.c.head_dim;
        const int64_t t = a.s.num_tokens;
        if (overlaps(d_q, q_token_stride, q_head_stride, t, q_heads, d, size, d_q_out, q_heads) ||
            overlaps(d_k, k_token_stride, k_head_stride, t, a.c.kv_heads, d, size, d_q_out, q_heads) ||
            overlaps(d_v, v_token_stride, v_head_stride, t, a.c.kv_heads, d, size, d_q_out, q_heads))
            return fail(LBQ_ERR_INVALID_ARG, "the rotated q must not overlap q, k or v");
    }
    a.k = {d_k, k_token_stride, k_head_stride};
    a.v = {d_v, v_token_stride, v_head_stride};
    a.q = {d_q, q_token_stride, q_head_stride};
    a.q_out = d_q_out;
    a.q_heads = q_heads;
    a.cos = d_cos;
    a.sin = d_sin;
    a.max_pos = max_pos;
    a.rot_dim = rot_dim;
    a.interleaved = interleaved != 0;
    a.max_new = step->max_new;
    const int64_t runs = (a.s.num_tokens >> a.c.log2_page) + 2 * (int64_t)a.s.batch;
    if (runs * a.c.kv_heads * 2 + 65536 >= (int64_t)1 << 24)  // (workgroups of 256 threads: below 2^32)
        return fail(LBQ_ERR_LIMIT, "%lld pages by %d heads in one append", (long long)runs, a.c.kv_heads);
    return launched(ctx, "append launch", [&] { return lbq::launch_kv_append(a, static_cast<hipStream_t>(stream)); });
}

static int attention_args(const lbq_kv_cache *cache, const lbq_kv_step *step, int32_t q_heads, lbq::KvAttention *a) {
    if (int e = check_cache(cache, &a->c)) return e;
    if (int e = check_step(step, false, &a->s)) return e;
    if (int e = check_query_heads(q_heads, a->c.kv_heads)) return e;
    a->q_heads = q_heads;
    const int64_t held = (int64_t)a->s.max_blocks * a->c.page_size;
    const int64_t longest = step->max_len ? std::min<int64_t>(step->max_len, held) : held;
    if (longest > MAX_LEN) return fail(LBQ_ERR_LIMIT, "sequences of %lld tokens", (long long)longest);
    a->max_len = (int)longest;
    a->max_new = step->max_new;
    if (step->num_tokens * q_heads > INT32_MAX)
        return fail(LBQ_ERR_LIMIT, "%lld tokens of %d heads in one call", (long long)step->num_tokens, q_heads);
    // (tiles of at least 128 rows, and one more for each sequence)
    if (step->num_tokens * q_heads / 128 + (int64_t)a->s.batch * a->c.kv_heads > lbq::MAX_GROUPS)
        return fail(LBQ_ERR_LIMIT, "%d sequences of %d heads and %lld tokens in one call", a->s.batch, a->c.kv_heads, (long long)step->num_tokens);
    return LBQ_OK;
}

int lbq_kv_attention_workspace(lbq_ctx *ctx, const lbq_kv_cache *cache, const lbq_kv_step *step, int32_t q_heads, size_t *bytes) {
    if (!ctx || !bytes) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_kv_attention_workspace");
    lbq::KvAttention a = {};
    if (int e = attention_args(cache, step, q_heads, &a)) return e;
    *bytes = 0;
    return launched(ctx, "workspace", [&] {
        *bytes = lbq::kv_attention_workspace(a);
        return hipSuccess;
    });
}

int lbq_kv_attention(lbq_ctx *ctx, const lbq_kv_cache *cache, const lbq_kv_step *step, uint32_t dtype, const void *d_q,
                     int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads, float scale, int32_t causal, int64_t window,
                     void *d_out, void *d_ws, size_t ws_bytes, void *stream) {
    if (!ctx) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_kv_attention");
    lbq::KvAttention a = {};
    if (int e = attention_args(cache, step, q_heads, &a)) return e;
    if (int e = check_dtype(dtype, &a.dtype)) return e;
    if (window < 0 || (window && !causal)) return fail(LBQ_ERR_SHAPE, "a window of %lld without a causal mask, or below 0", (long long)window);
    if (a.s.num_tokens == 0) return LBQ_OK;
    if (int e = check_rows("q", d_q, q_token_stride, q_head_stride, a.dtype)) return e;
    if (int e = check_rows("out", d_out, 0, 0, a.dtype)) return e;
    if (overlaps(d_q, q_token_stride, q_head_stride, a.s.num_tokens, q_heads, a.c.head_dim, a.dtype == lbq::DT_F32 ? 4 : 2, d_out, q_heads))
        return fail(LBQ_ERR_INVALID_ARG, "out must not overlap q");
    if (!aligned(d_ws, 16)) return fail(LBQ_ERR_INVALID_ARG, "the workspace must be 16-byte aligned");
    a.cu_q = a.s.cu;
    a.num_q = a.s.num_tokens;
    a.q = {d_q, q_token_stride, q_head_stride};
    a.out = d_out;
    a.scale = scale;
    a.causal = causal != 0;
    a.window = (int)std::min(window, MAX_LEN);  // (as wide as any sequence)
    a.ws = d_ws;
    a.ws_bytes = d_ws ? ws_bytes : 0;
    return launched(ctx, "attention launch", [&] { return lbq::launch_kv_attention(a, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
