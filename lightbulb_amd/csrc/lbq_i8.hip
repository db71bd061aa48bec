// lbq_i8.hip -- values to 8-bit codes by token, and the residual stream's update with the norms
// before and after a block.
#include "lbq_i8.hpp"

#include <algorithm>

namespace lbq {
namespace {

// TPR threads have a row, NV pieces of eight values each: piece threadIdx + j TPR.  One row a
// workgroup, or 256 / TPR of them.
template <int TPR>
struct RowShape {
    static constexpr int THREADS = TPR < 256 ? 256 : TPR, ROWS = THREADS / TPR, WAVES = TPR / 64;
};

template <typename V, typename F>
__device__ __forceinline__ V wave_all(V v, F f) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = f(v, __shfl_xor(v, d));
    return v;
}
// over the row's threads, in one order; `part` is this reduction's own
template <int WAVES, typename V, typename F>
__device__ __forceinline__ V row_all(V v, V *part, F f) {
    v = wave_all(v, f);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v = f(v, part[w]);
    }
    return v;
}
struct Sum {
    __device__ double operator()(double a, double b) const { return a + b; }
};
struct Max {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};

template <int DT>
constexpr int SIZE = DT == I8_F32 ? 4 : 2;

// Codes and scale of each row.  Bound by memory: a row is read once and held in registers (NV = 0: of
// rows wider than 65536, read twice, the second time out of the L2).
template <int DT, int TPR, int NV>
__global__ __launch_bounds__(RowShape<TPR>::THREADS) void k_i8_quantize(const void *__restrict__ x, int64_t stride, int64_t m, int k,
                                                                        int kp, int8_t *__restrict__ codes, float *__restrict__ scales) {
    using S = RowShape<TPR>;
    __shared__ uint32_t part[S::THREADS / 64];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * S::ROWS + threadIdx.x / TPR;
    if (S::ROWS > 1 && row >= m) return;  // (a whole wave, and no barrier follows)
    const char *xr = static_cast<const char *>(x) + row * stride * SIZE<DT>;
    int8_t *cr = codes + row * kp;
    uint32_t top = 0;
    float v[NV ? NV : 1][8];
    auto look = [&](const float *u) {
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, i8_magnitude(u[e]));
    };
    auto put = [&](int i, const float *u, float s, float inv) {
        uint32_t c[2];
        i8_codes8(u, s, inv, s > 0.f, c);
        *reinterpret_cast<uint2 *>(cr + i) = make_uint2(c[0], c[1]);
    };
    if constexpr (NV) {
#pragma unroll
        for (int j = 0; j < NV; j++) i8_load8<DT>(xr, 8 * (t + j * TPR), k, v[j]);
#pragma unroll
        for (int j = 0; j < NV; j++) look(v[j]);
    } else {
        for (int i = 8 * t; i < k; i += 8 * TPR) i8_load8<DT>(xr, i, k, v[0]), look(v[0]);
    }
    const float s = i8_scale(__uint_as_float(row_all<S::WAVES>(top, part, Max{}))), inv = 1.f / s;
    if (t == 0) scales[row] = s;
    if constexpr (NV) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (8 * (t + j * TPR) < kp) put(8 * (t + j * TPR), v[j], s, inv);
    } else {
        for (int i = 8 * t; i < kp; i += 8 * TPR) i8_load8<DT>(xr, i, k, v[0]), put(i, v[0], s, inv);
    }
}

// r = residual + scale gate post(x), y = pre(r), of a row: with u a row,
//   root mean square   u / sqrt(mean(u^2) + eps) (w + offset) + b
//   layer              (u - mean(u)) / sqrt(mean((u - mean(u))^2) + eps) (w + offset) + b
// in 64 bits throughout, which this machine has at the rate of 32: a value is rounded once, where it is
// stored, r as pre sees it not at all, and a code does not go by the order of a sum.  y as codes is
// rounded to f32 first.  Every value of a row is read before one is written.
template <int DX, int DR, int TPR, int NV>
__global__ __launch_bounds__(RowShape<TPR>::THREADS) void k_residual_norm(ResidualNorm a) {
    using S = RowShape<TPR>;
    __shared__ double sums[4][S::THREADS / 64];
    __shared__ uint32_t part[S::THREADS / 64];
    const int t = threadIdx.x % TPR, k = a.k;
    const int64_t row = (int64_t)blockIdx.x * S::ROWS + threadIdx.x / TPR;
    if (S::ROWS > 1 && row >= a.m) return;  // (a whole wave, and no barrier follows)
    double v[NV][8];
    auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < NV; j++) f(8 * (t + j * TPR), v[j]);
    };
    auto normed = [&](const NormArgs &n, int at) {
        if (!n.kind) return;
        double mean = 0, ss = 0;
        if (n.kind == 2) {
            each([&](int, const double *u) {
#pragma unroll
                for (int e = 0; e < 8; e++) mean += u[e];  // (zero behind the row's end)
            });
            mean = row_all<S::WAVES>(mean, sums[at], Sum{}) / k;
        }
        each([&](int i, double *u) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                u[e] = i + e < k ? u[e] - mean : 0.0;
                ss = fma(u[e], u[e], ss);
            }
        });
        const double inv = 1.0 / sqrt(row_all<S::WAVES>(ss, sums[at + 1], Sum{}) / k + (double)n.eps);
        each([&](int i, double *u) {
            if (i >= k) return;
            float w[8], b[8] = {};
            i8_load8<I8_F32>(n.w, i, k, w);
            if (n.b) i8_load8<I8_F32>(n.b, i, k, b);
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = fma(u[e] * inv, (double)w[e] + (double)n.offset, (double)b[e]);
        });
    };
    const char *xr = static_cast<const char *>(a.x.p) + row * a.x.stride * SIZE<DX>;
    float f[8];
    each([&](int i, double *u) {
        i8_load8<DX>(xr, i, k, f);
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = f[e];
    });
    normed(a.post, 0);
    if (a.gate.p) {
        const char *gr = static_cast<const char *>(a.gate.p) + row * a.gate.stride * SIZE<DX>;
        each([&](int i, double *u) {
            i8_load8<DX>(gr, i, k, f);
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] *= f[e];
        });
    }
    if (a.residual.p) {
        const char *rr = static_cast<const char *>(a.residual.p) + row * a.residual.stride * SIZE<DR>;
        each([&](int i, double *u) {
            i8_load8<DR>(rr, i, k, f);
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = fma(u[e], (double)a.scale, (double)f[e]);
        });
    } else if (a.scale != 1.f) {
        each([&](int, double *u) {
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] *= (double)a.scale;
        });
    }
    if (a.r) {
        char *out = static_cast<char *>(a.r) + row * k * SIZE<DR>;
        each([&](int i, const double *u) {
            if (i >= k) return;
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = (float)u[e];
            i8_store8<DR>(out, i, k, f);
        });
    }
    if (!a.pre.kind) return;
    normed(a.pre, 2);
    if (a.y) {
        char *out = static_cast<char *>(a.y) + row * k * SIZE<DX>;
        each([&](int i, const double *u) {
            if (i >= k) return;
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = (float)u[e];
            i8_store8<DX>(out, i, k, f);
        });
    } else {
        const int kp = (k + 127) / 128 * 128;
        uint32_t top = 0;
        each([&](int i, const double *u) {
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, i + e < k ? i8_magnitude((float)u[e]) : 0u);
        });
        const float s = i8_scale(__uint_as_float(row_all<S::WAVES>(top, part, Max{}))), inv = 1.f / s;
        if (t == 0) a.codes.scales[row] = s;
        int8_t *cr = a.codes.codes + row * kp;
        each([&](int i, const double *u) {
            if (i >= kp) return;
            uint32_t c[2];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = i + e < k ? (float)u[e] : 0.f;
            i8_codes8(f, s, inv, s > 0.f, c);
            *reinterpret_cast<uint2 *>(cr + i) = make_uint2(c[0], c[1]);
        });
    }
}

template <int DT, int TPR, int NV>
hipError_t quantize(const I8Rows &x, int64_t m, int k, int kp, const I8Tokens &t, hipStream_t st) {
    using S = RowShape<TPR>;
    k_i8_quantize<DT, TPR, NV><<<(unsigned)((m + S::ROWS - 1) / S::ROWS), S::THREADS, 0, st>>>(x.p, x.stride, m, k, kp, t.codes, t.scales);
    return hipGetLastError();
}
template <int DT>
hipError_t quantize_rows(const I8Rows &x, int64_t m, int k, const I8Tokens &t, hipStream_t st) {
    const int kp = (int)i8_kp(k);
    if (kp <= 512) return quantize<DT, 64, 1>(x, m, k, kp, t, st);
    if (kp <= 2048) return quantize<DT, 256, 1>(x, m, k, kp, t, st);
    if (kp <= 4096) return quantize<DT, 256, 2>(x, m, k, kp, t, st);
    if (kp <= 8192) return quantize<DT, 256, 4>(x, m, k, kp, t, st);
    if (kp <= 16384) return quantize<DT, 1024, 2>(x, m, k, kp, t, st);
    if (kp <= 65536) return quantize<DT, 1024, 8>(x, m, k, kp, t, st);
    return quantize<DT, 1024, 0>(x, m, k, kp, t, st);
}

template <int DX, int DR, int TPR, int NV>
hipError_t norm(const ResidualNorm &a, hipStream_t st) {
    using S = RowShape<TPR>;
    k_residual_norm<DX, DR, TPR, NV><<<(unsigned)((a.m + S::ROWS - 1) / S::ROWS), S::THREADS, 0, st>>>(a);
    return hipGetLastError();
}
template <int DX, int DR>
hipError_t norm_rows(const ResidualNorm &a, hipStream_t st) {
    const int kp = (int)i8_kp(a.k);
    if (kp <= 512) return norm<DX, DR, 64, 1>(a, st);
    if (kp <= 2048) return norm<DX, DR, 256, 1>(a, st);
    if (kp <= 8192) return norm<DX, DR, 512, 2>(a, st);
    if (kp <= 16384) return norm<DX, DR, 1024, 2>(a, st);
    return norm<DX, DR, 1024, 4>(a, st);
}
template <int DX>
hipError_t norm_stream(const ResidualNorm &a, hipStream_t st) {
    return a.residual.dtype == I8_F32 ? norm_rows<DX, I8_F32>(a, st)
         : a.residual.dtype == I8_F16 ? norm_rows<DX, I8_F16>(a, st)
                                      : norm_rows<DX, I8_BF16>(a, st);
}

}  // namespace

hipError_t launch_i8_quantize(const I8Rows &x, int64_t m, int64_t k, const I8Tokens &t, hipStream_t st) {
    return x.dtype == I8_F32 ? quantize_rows<I8_F32>(x, m, (int)k, t, st)
         : x.dtype == I8_F16 ? quantize_rows<I8_F16>(x, m, (int)k, t, st)
                             : quantize_rows<I8_BF16>(x, m, (int)k, t, st);
}

hipError_t launch_residual_norm(const ResidualNorm &a, hipStream_t st) {
    return a.x.dtype == I8_F32 ? norm_stream<I8_F32>(a, st) : a.x.dtype == I8_F16 ? norm_stream<I8_F16>(a, st) : norm_stream<I8_BF16>(a, st);
}

}  // namespace lbq
