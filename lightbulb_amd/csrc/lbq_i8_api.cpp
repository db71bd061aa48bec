// lbq_i8_api.cpp -- C entry points of the 8-bit integer linears and of the norms between them
// (include/lbq.h): the arguments' checks and the launches.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/lbq.h"
#include "lbq_i8.hpp"

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
int size_of(int dt) { return dt == lbq::I8_F32 ? 4 : 2; }

bool overlap(const void *a, int64_t an, const void *b, int64_t bn) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p && q && p < q + (uintptr_t)bn && q < p + (uintptr_t)an;
}

int check_type(const char *what, uint32_t t, int *dt) {
    *dt = t == LBQ_TYPE_F32 ? lbq::I8_F32 : t == LBQ_TYPE_F16 ? lbq::I8_F16 : lbq::I8_BF16;
    if (t != LBQ_TYPE_F32 && t != LBQ_TYPE_F16 && t != LBQ_TYPE_BF16)
        return fail(LBQ_ERR_UNSUPPORTED_TYPE, "type %u of %s is none of F32, F16 and BF16", t, what);
    return LBQ_OK;
}

int check_sizes(int64_t m, int64_t k, int64_t most_k) {
    if (m < 0 || k < 1) return fail(LBQ_ERR_SHAPE, "%lld rows of %lld values", (long long)m, (long long)k);
    if (m > lbq::I8_MAX_M || k > most_k)
        return fail(LBQ_ERR_LIMIT, "%lld rows of %lld values exceed %lld of %lld", (long long)m, (long long)k, (long long)lbq::I8_MAX_M, (long long)most_k);
    return LBQ_OK;
}

int check_rows(const char *what, const void *p, int64_t stride, int64_t k, int dt, lbq::I8Rows *rows) {
    if (!p) return fail(LBQ_ERR_INVALID_ARG, "null %s", what);
    if (!aligned(p, size_of(dt))) return fail(LBQ_ERR_INVALID_ARG, "%s must be aligned to its elements", what);
    if (stride < 0 || stride > (int64_t)1 << 38) return fail(LBQ_ERR_SHAPE, "rows of %s %lld values apart", what, (long long)stride);
    *rows = {p, stride, dt};
    return LBQ_OK;
}
int64_t bytes_of(const lbq::I8Rows &r, int64_t m, int64_t k) { return r.p ? ((m - 1) * r.stride + k) * size_of(r.dtype) : 0; }

int check_tokens(const void *codes, const void *scales, int64_t m, int64_t k, lbq::I8Tokens *t) {
    if (!codes || !scales) return fail(LBQ_ERR_INVALID_ARG, "null codes or scales of the tokens");
    if (!aligned(codes, 16)) return fail(LBQ_ERR_INVALID_ARG, "the tokens' codes must be 16-byte aligned");
    if (!aligned(scales, 4)) return fail(LBQ_ERR_INVALID_ARG, "the tokens' scales must be 4-byte aligned");
    if (overlap(codes, m * lbq::i8_kp(k), scales, m * 4)) return fail(LBQ_ERR_INVALID_ARG, "the tokens' codes and scales must not overlap");
    *t = {static_cast<int8_t *>(const_cast<void *>(codes)), static_cast<float *>(const_cast<void *>(scales))};
    return LBQ_OK;
}

int check_weight(const lbq_i8_weight *w, int i, lbq::I8Linear *a) {
    if (!w || !w->d_codes || !w->d_scales) return fail(LBQ_ERR_INVALID_ARG, "null weight, codes or scales");
    if (!aligned(w->d_codes, 16)) return fail(LBQ_ERR_INVALID_ARG, "a weight's codes must be 16-byte aligned");
    if (!aligned(w->d_scales, 4) || !aligned(w->d_bias, 4)) return fail(LBQ_ERR_INVALID_ARG, "a weight's scales and bias must be 4-byte aligned");
    if (w->n < 1) return fail(LBQ_ERR_SHAPE, "a weight of %lld channels", (long long)w->n);
    if (w->n > lbq::I8_MAX_N) return fail(LBQ_ERR_LIMIT, "a weight of %lld channels exceeds %lld", (long long)w->n, (long long)lbq::I8_MAX_N);
    a->w[i] = w->d_codes, a->t[i] = w->d_scales, a->bias[i] = w->d_bias, a->n[i] = (int)w->n;
    return LBQ_OK;
}

// whether [p, p + bytes) meets a weight's memory
bool over_weights(const void *p, int64_t bytes, const lbq::I8Linear &a) {
    for (int i = 0; i < a.count; i++)
        if (overlap(p, bytes, a.w[i], (int64_t)a.n[i] * a.kp) || overlap(p, bytes, a.t[i], (int64_t)a.n[i] * 4) || overlap(p, bytes, a.bias[i], (int64_t)a.n[i] * 4))
            return true;
    return false;
}

// everything but the outputs; *quantize: the values need a launch of their own
int linear_args(uint32_t x_type, const void *d_x, int64_t x_stride, void *d_codes, float *d_scales, int64_t m, int64_t k,
                const lbq_i8_weight *const *ws, int count, uint32_t out_type, lbq::I8Linear *a, bool *quantize) {
    if (!ws) return fail(LBQ_ERR_INVALID_ARG, "null weights");
    if (int e = check_sizes(m, k, lbq::I8_MAX_K)) return e;
    int64_t rows = 0;
    for (int i = 0; i < count; i++) {
        if (int e = check_weight(ws[i], i, a)) return e;
        rows += ws[i]->n;
    }
    // (tiles take a thread for 16 outputs at most, streams of few tokens 32 threads a channel: with each weight's last tiles, which
    // need not be full, a launch stays below 2^32 threads)
    if (m * rows >= lbq::I8_MAX_OUTPUTS)
        return fail(LBQ_ERR_LIMIT, "%lld tokens by %lld channels in one call", (long long)m, (long long)rows);
    if (int e = check_type("the outputs", out_type, &a->out)) return e;
    a->m = m, a->k = (int)k, a->kp = (int)lbq::i8_kp(k), a->count = count;
    *quantize = false;
    if (m == 0) return LBQ_OK;
    lbq::I8Tokens t = {};
    if (d_x) {
        int dt;
        if (int e = check_type("x", x_type, &dt)) return e;
        if (int e = check_rows("x", d_x, x_stride, k, dt, &a->x)) return e;
        *quantize = !lbq::i8_quantizes_in_kernel(m, k, rows);
    }
    if (!d_x || *quantize)
        if (int e = check_tokens(d_codes, d_scales, m, k, &t)) return e;
    if (*quantize && (overlap(d_x, bytes_of(a->x, m, k), t.codes, m * a->kp) || overlap(d_x, bytes_of(a->x, m, k), t.scales, m * 4)))
        return fail(LBQ_ERR_INVALID_ARG, "the codes' memory must not overlap x");
    if (*quantize && (over_weights(t.codes, m * a->kp, *a) || over_weights(t.scales, m * 4, *a)))
        return fail(LBQ_ERR_INVALID_ARG, "the codes' memory must not overlap a weight");
    a->codes = t.codes, a->scales = t.scales;
    return LBQ_OK;
}

int check_output(void *y, int i, int64_t n, lbq::I8Linear *a) {
    const int size = size_of(a->out);
    if (!y) return fail(LBQ_ERR_INVALID_ARG, "null output");
    if (!aligned(y, size)) return fail(LBQ_ERR_INVALID_ARG, "an output must be aligned to its elements");
    const int64_t bytes = a->m * n * size;
    if (overlap(y, bytes, a->codes, a->m * a->kp) || overlap(y, bytes, a->scales, a->m * 4) || overlap(y, bytes, a->x.p, bytes_of(a->x, a->m, a->k)))
        return fail(LBQ_ERR_INVALID_ARG, "an output must not overlap the input");
    if (over_weights(y, bytes, *a)) return fail(LBQ_ERR_INVALID_ARG, "an output must not overlap a weight");
    for (int j = 0; j < i; j++)
        if (overlap(y, bytes, a->y[j], a->m * a->n[j] * size)) return fail(LBQ_ERR_INVALID_ARG, "the outputs must not overlap");
    a->y[i] = y;
    return LBQ_OK;
}

int run_linear(lbq_ctx *ctx, lbq::I8Linear &a, bool quantize, void *stream) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return launched(ctx, "integer linear launch", [&] {
        if (quantize) {
            const hipError_t e = lbq::launch_i8_quantize(a.x, a.m, a.k, {const_cast<int8_t *>(a.codes), const_cast<float *>(a.scales)}, st);
            if (e != hipSuccess) return e;
            a.x.p = nullptr;
        }
        return lbq::launch_i8_linear(a, st);
    });
}

int check_norm(const char *what, const lbq_norm *n, lbq::NormArgs *a) {
    *a = {};
    if (!n) return LBQ_OK;
    if (n->kind != LBQ_NORM_RMS && n->kind != LBQ_NORM_LAYER)
        return fail(LBQ_ERR_UNSUPPORTED_TYPE, "kind %d of the %s norm is neither root mean square (0) nor layer (1)", n->kind, what);
    if (!n->d_weight) return fail(LBQ_ERR_INVALID_ARG, "null weight of the %s norm", what);
    if (!aligned(n->d_weight, 4) || !aligned(n->d_bias, 4)) return fail(LBQ_ERR_INVALID_ARG, "the %s norm's weight and bias must be 4-byte aligned", what);
    if (!(n->eps >= 0)) return fail(LBQ_ERR_SHAPE, "eps %g of the %s norm", n->eps, what);
    *a = {n->kind + 1, n->eps, n->offset, n->d_weight, n->d_bias};
    return LBQ_OK;
}

}  // namespace

extern "C" {

int lbq_i8_quantize(lbq_ctx *ctx, uint32_t type, const void *d_x, int64_t row_stride, int64_t m, int64_t k, int8_t *d_codes,
                    float *d_scales, void *stream) {
    if (!ctx) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_i8_quantize");
    int dt;
    lbq::I8Rows x;
    lbq::I8Tokens t;
    if (int e = check_type("x", type, &dt)) return e;
    if (int e = check_sizes(m, k, lbq::I8_MAX_K)) return e;
    if (m == 0) return LBQ_OK;
    if (int e = check_rows("x", d_x, row_stride, k, dt, &x)) return e;
    if (int e = check_tokens(d_codes, d_scales, m, k, &t)) return e;
    if (overlap(d_x, bytes_of(x, m, k), d_codes, m * lbq::i8_kp(k)) || overlap(d_x, bytes_of(x, m, k), d_scales, m * 4))
        return fail(LBQ_ERR_INVALID_ARG, "the codes' memory must not overlap x");
    return launched(ctx, "quantise launch", [&] { return lbq::launch_i8_quantize(x, m, k, t, static_cast<hipStream_t>(stream)); });
}

int lbq_i8_linear(lbq_ctx *ctx, uint32_t x_type, const void *d_x, int64_t x_stride, int8_t *d_codes, float *d_scales, int64_t m,
                  int64_t k, const lbq_i8_weight *const *ws, int count, uint32_t out_type, void *const *d_ys, void *stream) {
    if (!ctx || !d_ys) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_i8_linear");
    if (count < 1 || count > LBQ_GROUP_MAX) return fail(LBQ_ERR_SHAPE, "between 1 and %d weights per call, got %d", LBQ_GROUP_MAX, count);
    lbq::I8Linear a = {};
    bool quantize;
    if (int e = linear_args(x_type, d_x, x_stride, d_codes, d_scales, m, k, ws, count, out_type, &a, &quantize)) return e;
    if (m == 0) return LBQ_OK;
    for (int i = 0; i < count; i++)
        if (int e = check_output(d_ys[i], i, a.n[i], &a)) return e;
    return run_linear(ctx, a, quantize, stream);
}

int lbq_i8_gate_up_silu(lbq_ctx *ctx, uint32_t x_type, const void *d_x, int64_t x_stride, int8_t *d_codes, float *d_scales, int64_t m,
                        int64_t k, const lbq_i8_weight *gate, const lbq_i8_weight *up, uint32_t out_type, void *d_y, void *stream) {
    if (!ctx) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_i8_gate_up_silu");
    const lbq_i8_weight *const ws[2] = {gate, up};
    lbq::I8Linear a = {};
    bool quantize;
    if (int e = linear_args(x_type, d_x, x_stride, d_codes, d_scales, m, k, ws, 2, out_type, &a, &quantize)) return e;
    if (a.n[0] != a.n[1]) return fail(LBQ_ERR_SHAPE, "gate of %d and up of %d channels", a.n[0], a.n[1]);
    if (m == 0) return LBQ_OK;
    if (int e = check_output(d_y, 0, a.n[0], &a)) return e;
    a.pair = true;
    return run_linear(ctx, a, quantize, stream);
}

int lbq_residual_norm(lbq_ctx *ctx, uint32_t type, const void *d_x, int64_t x_stride, uint32_t residual_type, const void *d_residual,
                      int64_t residual_stride, const lbq_norm *post, const void *d_gate, int64_t gate_stride, float scale,
                      const lbq_norm *norm, int64_t m, int64_t k, void *d_r, void *d_y, int8_t *d_codes, float *d_scales, void *stream) {
    if (!ctx) return fail(LBQ_ERR_INVALID_ARG, "null argument to lbq_residual_norm");
    lbq::ResidualNorm a = {};
    int dt, rt;
    if (int e = check_type("x", type, &dt)) return e;
    if (int e = check_type("the residual", residual_type, &rt)) return e;
    if (int e = check_sizes(m, k, lbq::NORM_MAX_K)) return e;
    if (int e = check_norm("first", post, &a.post)) return e;
    if (int e = check_norm("second", norm, &a.pre)) return e;
    if (m == 0) return LBQ_OK;
    if (int e = check_rows("x", d_x, x_stride, k, dt, &a.x)) return e;
    a.residual.dtype = rt;
    if (d_residual)
        if (int e = check_rows("the residual", d_residual, residual_stride, k, rt, &a.residual)) return e;
    if (d_gate)
        if (int e = check_rows("the gate", d_gate, gate_stride, k, dt, &a.gate)) return e;
    if (d_codes || d_scales) {
        if (d_y || !norm) return fail(LBQ_ERR_INVALID_ARG, "codes are the second norm's result in the place of y");
        if (int e = check_tokens(d_codes, d_scales, m, k, &a.codes)) return e;
    } else if (!!norm != !!d_y) {
        return fail(LBQ_ERR_INVALID_ARG, "a second norm and its result go together");
    }
    if (!d_r && !norm) return fail(LBQ_ERR_INVALID_ARG, "no result is wanted");
    if (!aligned(d_r, size_of(rt)) || !aligned(d_y, size_of(dt))) return fail(LBQ_ERR_INVALID_ARG, "the results must be aligned to their elements");
    // (a row's values are all read before one is written: r may take the residual's place, row for row)
    const bool in_place = d_r && d_r == d_residual && (residual_stride == k || m == 1);
    const struct { const void *p; int64_t n; } out[4] = {{d_r, m * k * size_of(rt)}, {d_y, m * k * size_of(dt)}, {d_codes, m * lbq::i8_kp(k)}, {d_scales, m * 4}};
    for (int i = 0; i < 4; i++) {
        if (overlap(out[i].p, out[i].n, d_x, bytes_of(a.x, m, k)) || overlap(out[i].p, out[i].n, d_gate, bytes_of(a.gate, m, k)) ||
            (!(i == 0 && in_place) && overlap(out[i].p, out[i].n, d_residual, bytes_of(a.residual, m, k))))
            return fail(LBQ_ERR_INVALID_ARG, "the results must not overlap the inputs");
        for (const lbq::NormArgs *n : {&a.post, &a.pre})
            if (overlap(out[i].p, out[i].n, n->w, k * 4) || overlap(out[i].p, out[i].n, n->b, k * 4))
                return fail(LBQ_ERR_INVALID_ARG, "the results must not overlap a norm's weight or bias");
        for (int j = 0; j < i; j++)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return fail(LBQ_ERR_INVALID_ARG, "the results must not overlap");
    }
    a.scale = scale, a.m = m, a.k = (int)k, a.r = d_r, a.y = d_y;
    return launched(ctx, "norm launch", [&] { return lbq::launch_residual_norm(a, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
