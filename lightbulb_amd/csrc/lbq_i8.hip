// lbq_i8.hip -- values to 8-bit codes by token, and the residual stream's update with the norms
// before and after a block.
#include "lbq_i8.hpp"

namespace lbq {
namespace {

// TPR threads have a row, NV pieces of eight values each: piece threadIdx + j TPR.  One row a
// workgroup, or 256 / TPR of them.
template <int TPR>
struct RowShape {
    static constexpr int THREADS = TPR < 128 ? 256 : TPR, ROWS = THREADS / TPR, WAVES = TPR / 64;
};

// over the row's threads, in one order; `part` is this reduction's own
template <int WAVES, typename V, typename F>
__device__ __forceinline__ V row_all(V v, V *part, F f) {
    v = i8_wave_all(v, f);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[threadIdx.x / 64 / WAVES * WAVES];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v = f(v, part[threadIdx.x / 64 / WAVES * WAVES + w]);
    }
    return v;
}
template <int DT>
constexpr int SIZE = DT == I8_F32 ? 4 : 2;

// Codes and scale of each row.  Bound by memory: a row is read once and held in registers (NV = 0: of
// rows wider than 65536, read twice, the second time out of the L2).  4096 rows of 14336 bf16 values 33 us, 5.3 TB/s of what is
// read and written; 2048 of 4096 f32 values 8.7 us, 4.8 TB/s; 16 of 14336 3.8 us, nearly all of it a launch, a load and a barrier.
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
    const float s = i8_scale(__uint_as_float(row_all<S::WAVES>(top, part, I8Max{}))), inv = 1.f / s;
    if (t == 0) scales[row] = s;
    if constexpr (NV) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (8 * (t + j * TPR) < kp) put(8 * (t + j * TPR), v[j], s, inv);
    } else {
        for (int i = 8 * t; i < kp; i += 8 * TPR) i8_load8<DT>(xr, i, k, v[0]), put(i, v[0], s, inv);
    }
}

// The sums that a norm needs of a row u, about a value c near it: sum of u - c and of its square.
struct Moments {
    double a, b;
};
template <int WAVES>
__device__ __forceinline__ Moments row_all(Moments v, Moments *part) {
    v.a = i8_wave_all(v.a, I8Sum{}), v.b = i8_wave_all(v.b, I8Sum{});
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v = {v.a + part[w].a, v.b + part[w].b};
    }
    return v;
}

// What a norm takes of a row: the mean in F and what F leaves of it, and 1 / sqrt(..).  In 32 bits a row of values whose
// inverse is near the ends of the range is lifted by a power of two first, and mean and inverse are those of the lifted row.
template <typename F>
struct NormOf {
    F mean = 0, left = 0, inv = 1, lift = 1;
    __device__ __forceinline__ void set(double m, double i) {
        if constexpr (sizeof(F) == 4) {
            lift = i > 0x1p100 ? 0x1p60f : i < 0x1p-100 ? 0x1p-60f : 1.f;
            lift = __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(lift)));
            m *= (double)lift, i /= (double)lift;
        }
        mean = (F)m, left = sizeof(F) == 4 ? (F)(m - (double)mean) : (F)0, inv = (F)i;
    }
    __device__ __forceinline__ F off(F u) const { return sizeof(F) == 4 ? (u - mean) - left : u - mean; }  // u - mean, off by two roundings of itself
};

// r = residual + scale gate post(x), y = pre(r), of a row: with u a row,
//   root mean square   u / sqrt(mean(u^2) + eps) (w + offset) + b
//   layer              (u - mean(u)) / sqrt(mean((u - mean(u))^2) + eps) (w + offset) + b
// Sums are in 64 bits.  Values are in F: 32 bits where y is a value, 64 where it becomes a code, which so does not go by the order
// of a sum (f32's last bits would turn one code in 10^5), rounded to f32 before it does.  A variance is formed in one pass, about the
// row's first value c: as the row holds c, (c - mean)^2 is at most k times the variance, and the difference of the sums loses no
// more than k 2^-53.  The row stays in registers as it was read, and r is formed anew for each pass over it: held in 64 bits it
// would take twice the registers, and with them go the rows that a CU has on the way.  Every value of a row is read before one
// is written (r may lie where residual does).
// Bound by memory: 4096 rows of 4096 bf16 values (x, stream, r, y) 28 us, 4.8 TB/s; the norms' own vectors come out of the L2 for
// every row, which is what 4000 rows of 5000 f16 with a gate and a layer norm of weight and bias pay for, 43 us for 33 with a weight alone.
// Two rows a workgroup, or workgroups that hold the vectors for row after row, have fewer rows on the way: 43 to 45 us.
// One row of 4096 takes 4.8 us: two reads one behind the other and two reductions.
template <int DX, int DR, int TPR, int NV, typename F>
__global__ __launch_bounds__(RowShape<TPR>::THREADS) void k_residual_norm(ResidualNorm a) {
    using S = RowShape<TPR>;
    static_assert(S::ROWS == 1 || S::WAVES == 1, "barriers of one row");
    __shared__ Moments sums[2][S::WAVES];
    __shared__ uint32_t part[S::WAVES];
    const int t = threadIdx.x % TPR, k = a.k;
    const int64_t row = (int64_t)blockIdx.x * S::ROWS + threadIdx.x / TPR;
    if (S::ROWS > 1 && row >= a.m) return;  // (a whole wave, and no barrier follows)
    const char *xr = static_cast<const char *>(a.x.p) + row * a.x.stride * SIZE<DX>;
    const char *gr = a.gate.p ? static_cast<const char *>(a.gate.p) + row * a.gate.stride * SIZE<DX> : nullptr;
    const char *rr = a.residual.p ? static_cast<const char *>(a.residual.p) + row * a.residual.stride * SIZE<DR> : nullptr;
    I8Piece<DX> x[NV], g[NV];
    I8Piece<DR> res[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = 8 * (t + j * TPR);
        if (i < k) {
            x[j] = i8_piece<DX>(xr, i, k);
            if (rr) res[j] = i8_piece<DR>(rr, i, k);
            if (gr) g[j] = i8_piece<DX>(gr, i, k);
        }
    }
    // (the row's first values, for c)
    const bool layer = a.post.kind == 2 || a.pre.kind == 2;
    const I8Piece<DX> x0 = layer ? i8_piece<DX>(xr, 0, 1) : I8Piece<DX>{};
    const I8Piece<DR> r0 = layer && rr ? i8_piece<DR>(rr, 0, 1) : I8Piece<DR>{};
    const I8Piece<DX> g0 = layer && gr ? i8_piece<DX>(gr, 0, 1) : I8Piece<DX>{};

    auto statistics = [&](const NormArgs &n, double c, Moments *at, NormOf<F> &of, auto values) {
        Moments s = {0, 0};
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = 8 * (t + j * TPR);
            if (i >= k) continue;
            F u[8];
            values(j, i, u);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const double d = i + e < k ? (double)u[e] - c : 0.0;
                s.a += d, s.b = fma(d, d, s.b);
            }
        }
        s = row_all<S::WAVES>(s, at);
        const double off = n.kind == 2 ? s.a / k : 0.0;
        const double var = fma(-off, off, s.b / k);
        of.set(n.kind == 2 ? c + off : 0.0, 1.0 / sqrt((var < 0 ? 0.0 : var) + (double)n.eps));  // (a NaN stays one)
    };
    // u -> (u - mean) inv (w + offset) + b
    auto scaled = [&](const NormArgs &n, const NormOf<F> &of, int i, F *u) {
        const I8Piece<I8_F32> w = i8_piece<I8_F32>(n.w, i, k);
        if (sizeof(F) == 4 && of.lift != 1) {
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] *= of.lift;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = of.off(u[e]) * of.inv * ((F)w[e] + (F)n.offset);
        if (n.b) {
            const I8Piece<I8_F32> b = i8_piece<I8_F32>(n.b, i, k);
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] += (F)b[e];
        }
    };
    NormOf<F> post, pre;
    auto stream = [&](const I8Piece<DX> &xv, const I8Piece<DX> &gv, const I8Piece<DR> &rv, int i, F *u) {
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = xv[e];
        if (a.post.kind) scaled(a.post, post, i, u);
        if (gr) {
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] *= (F)gv[e];
        }
        if (rr) {
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = __builtin_elementwise_fma(u[e], (F)a.scale, (F)rv[e]);
        } else if (a.scale != 1.f) {
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] *= (F)a.scale;
        }
    };
    if (a.post.kind) {
        statistics(a.post, a.post.kind == 2 ? (double)x0[0] : 0.0, sums[0], post, [&](int j, int, F *u) {
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = x[j][e];
        });
    }
    if (a.pre.kind) {
        double c = 0;
        if (a.pre.kind == 2) {
            F u[8];
            stream(x0, g0, r0, 0, u);
            c = u[0];
        }
        statistics(a.pre, c, sums[1], pre, [&](int j, int i, F *u) { stream(x[j], g[j], res[j], i, u); });
    }
    const int kp = (k + 127) / 128 * 128;
    uint32_t top = 0;
    float y[NV][8];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = 8 * (t + j * TPR);
#pragma unroll
        for (int e = 0; e < 8; e++) y[j][e] = 0.f;
        if (i >= k) continue;
        F u[8];
        stream(x[j], g[j], res[j], i, u);
        if (a.r) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = (float)u[e];
            i8_store8<DR>(static_cast<char *>(a.r) + row * k * SIZE<DR>, i, k, f);
        }
        if (!a.pre.kind) continue;
        scaled(a.pre, pre, i, u);
#pragma unroll
        for (int e = 0; e < 8; e++) y[j][e] = i + e < k ? (float)u[e] : 0.f;
        if constexpr (sizeof(F) == 4) {
            i8_store8<DX>(static_cast<char *>(a.y) + row * k * SIZE<DX>, i, k, y[j]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, i8_magnitude(y[j][e]));
        }
    }
    if constexpr (sizeof(F) == 8) {
        const float s = i8_scale(__uint_as_float(row_all<S::WAVES>(top, part, I8Max{}))), is = 1.f / s;
        if (t == 0) a.codes.scales[row] = s;
        int8_t *cr = a.codes.codes + row * kp;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = 8 * (t + j * TPR);
            uint32_t c[2];
            i8_codes8(y[j], s, is, s > 0.f, c);
            if (i < kp) *reinterpret_cast<uint2 *>(cr + i) = make_uint2(c[0], c[1]);
        }
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
    if (kp <= 4096) return quantize<DT, 512, 1>(x, m, k, kp, t, st);
    if (kp <= 8192) return quantize<DT, 512, 2>(x, m, k, kp, t, st);
    // (14336 bf16 values: 16 rows 3.8 us, with 512 threads 4.3; 4096 rows 35.4 and 32.9)
    if (kp <= 16384) return m <= 512 ? quantize<DT, 1024, 2>(x, m, k, kp, t, st) : quantize<DT, 512, 4>(x, m, k, kp, t, st);
    if (kp <= 65536) return quantize<DT, 1024, 8>(x, m, k, kp, t, st);
    return quantize<DT, 1024, 0>(x, m, k, kp, t, st);
}

template <int DX, int DR, int TPR, int NV>
hipError_t norm(const ResidualNorm &a, hipStream_t st) {
    using S = RowShape<TPR>;
    const unsigned blocks = (unsigned)((a.m + S::ROWS - 1) / S::ROWS);
    if (a.codes.codes) k_residual_norm<DX, DR, TPR, NV, double><<<blocks, S::THREADS, 0, st>>>(a);
    else k_residual_norm<DX, DR, TPR, NV, float><<<blocks, S::THREADS, 0, st>>>(a);
    return hipGetLastError();
}
template <int DX, int DR>
hipError_t norm_rows(const ResidualNorm &a, hipStream_t st) {
    const int kp = (int)i8_kp(a.k);
    // (the fewest threads that leave a thread few pieces: 30000 rows of 512 24 us, with 256 threads 46; 8000 of 2048 26, with
    // 512 threads 34; 4000 of 5000 43, with 512 46)
    if (kp <= 512) return norm<DX, DR, 64, 1>(a, st);
    if (kp <= 2048) return norm<DX, DR, 256, 1>(a, st);
    if (kp <= 4096) return norm<DX, DR, 512, 1>(a, st);
    if (kp <= 6144) return norm<DX, DR, 256, 3>(a, st);
    if (kp <= 8192) return norm<DX, DR, 512, 2>(a, st);
    // (16-bit values of 14336 with codes: 64 rows 14.7 us, with 512 threads 15.8; 1400 rows 53.9 and 48.0, with a first norm 93.7 and
    // 75.5; 2048 of 10000 58.8 and 47.8.  f32, whose pieces are twice the registers, 79.6 and 85.5.  With the threads the order of a
    // row's sums changes: a value's last bit may go by whether m is above 256 there)
    if constexpr (DX != I8_F32) {
        if (kp <= 12288 && a.m > 256) return norm<DX, DR, 512, 3>(a, st);
        if (kp <= 16384 && a.m > 256) return norm<DX, DR, 512, 4>(a, st);
    }
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
