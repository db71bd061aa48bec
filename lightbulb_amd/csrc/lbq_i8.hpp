// lbq_i8.hpp -- linears in 8-bit integers with a scale for each token and channel, and the norms
// between them: what their kernels and their C entry points share.
//
// A row of codes has kp = k rounded up to 128 bytes, zeros from k on, so that every kernel reads
// whole 16-byte pieces and no width is a special case.  Sums of code products are int32 and exact:
// k is at most 131071, below which 2^14 k < 2^31.  So a result does not go by the order of the sum,
// by the tile that it falls into or by the rows beside it.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

namespace lbq {

enum : int { I8_F32 = 0, I8_F16 = 1, I8_BF16 = 2 };
constexpr int I8_GROUP = 4;
constexpr int64_t I8_MAX_K = 131071, I8_MAX_N = (int64_t)1 << 24, I8_MAX_M = ((int64_t)1 << 22) - 1;  // (workgroups of up to 1024 threads: below 2^32)
constexpr int64_t I8_MAX_OUTPUTS = (int64_t)1 << 35;  // tokens times channels of a call stay below
constexpr int64_t NORM_MAX_K = 32768;
constexpr int I8_FUSED_ROWS = 4, I8_FUSED_CODES = 16384, I8_FUSED_CHANNELS = 16384;
inline int64_t i8_kp(int64_t k) { return (k + 127) / 128 * 128; }

// rows of values [m][k], `stride` elements apart
struct I8Rows {
    const void *p;
    int64_t stride;
    int dtype;
};
struct I8Tokens {
    int8_t *codes;  // [m][kp]
    float *scales;  // [m]
};

hipError_t launch_i8_quantize(const I8Rows &x, int64_t m, int64_t k, const I8Tokens &t, hipStream_t st);

// products of one set of tokens with up to I8_GROUP weights, or of a gate/up pair
struct I8Linear {
    const int8_t *codes;  // [m][kp]
    const float *scales;
    int64_t m;
    int k, kp, count;
    bool pair;  // weights 0 and 1: y[0] = silu(x . w0) * (x . w1)
    int out;    // I8_F32, ..
    const int8_t *w[I8_GROUP];  // [n][kp]
    const float *t[I8_GROUP], *bias[I8_GROUP];
    void *y[I8_GROUP];  // [m][n]
    int n[I8_GROUP];
    I8Rows x;  // values that the kernel quantises itself (x.p nullptr: codes and scales are there)
};
// whether the product's kernel quantises m rows of values itself; channels: of all its weights
bool i8_quantizes_in_kernel(int64_t m, int64_t k, int64_t channels);
bool i8_streams(const I8Linear &a);  // the kernel for few tokens
hipError_t launch_i8_stream(const I8Linear &a, hipStream_t st);
hipError_t launch_i8_linear(const I8Linear &a, hipStream_t st);

struct NormArgs {
    int kind;  // 0: none, 1: root mean square, 2: layer
    float eps, offset;
    const float *w, *b;
};
struct ResidualNorm {
    I8Rows x, residual, gate;  // residual.p, gate.p: may be nullptr; gate.stride 0: one row for all
    NormArgs post, pre;
    float scale;
    int64_t m;
    int k;
    void *r, *y;  // [m][k]; r in residual's type, y in x's; nullptr: not wanted
    I8Tokens codes;
};
hipError_t launch_residual_norm(const ResidualNorm &a, hipStream_t st);

#ifdef __HIPCC__
// eight values from element i on of a row of k, zero behind its end; rows need no more than their
// elements' alignment
template <int DT>
struct I8Piece {
    uint32_t u[DT == I8_F32 ? 8 : 4];
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (DT == I8_F32) return __uint_as_float(u[e]);
        const uint32_t b = e & 1 ? u[e >> 1] >> 16 : u[e >> 1] & 0xffffu;
        return DT == I8_BF16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half((unsigned short)b));
    }
};
template <int DT>
__device__ __forceinline__ I8Piece<DT> i8_piece(const void *row, int i, int k) {
    I8Piece<DT> v;
    if constexpr (DT == I8_F32) {
        struct __attribute__((packed, aligned(4))) V { uint32_t u[8]; };
        const uint32_t *p = static_cast<const uint32_t *>(row) + i;
        if (i + 8 <= k) {
            const V w = *reinterpret_cast<const V *>(p);
#pragma unroll
            for (int e = 0; e < 8; e++) v.u[e] = w.u[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v.u[e] = i + e < k ? p[e] : 0u;
        }
    } else {
        typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
        const uint16_t *p = static_cast<const uint16_t *>(row) + i;
        if (i + 8 <= k) {
            const u32x4a2 w = *reinterpret_cast<const u32x4a2 *>(p);
#pragma unroll
            for (int e = 0; e < 4; e++) v.u[e] = w[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                v.u[e] = (i + 2 * e < k ? p[2 * e] : 0u) | (i + 2 * e + 1 < k ? (uint32_t)p[2 * e + 1] << 16 : 0u);
        }
    }
    return v;
}
template <int DT>
__device__ __forceinline__ void i8_load8(const void *row, int i, int k, float v[8]) {
    const I8Piece<DT> p = i8_piece<DT>(row, i, k);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = p[e];
}

// an f32 value as it is: without this the compiler forms some F16 results from the product itself, in one rounding for
// two, and the same output would go by the kernel that it comes from
__device__ __forceinline__ float i8_f32(float v) {
    asm("" : "+v"(v));
    return v;
}
// rounded to nearest even
template <int DT>
__device__ __forceinline__ uint32_t i8_bits16(float v) {
    if constexpr (DT == I8_F16) v = i8_f32(v);
    if constexpr (DT == I8_F16) return __half_as_ushort(__float2half_rn(v));
    return __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <int DT>
__device__ __forceinline__ void i8_store(void *p, int64_t i, float v) {
    if constexpr (DT == I8_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)i8_bits16<DT>(v);
}
template <int DT>
__device__ __forceinline__ void i8_store8(void *row, int i, int k, const float v[8]) {
    if (i + 8 > k) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (i + e < k) i8_store<DT>(row, i + e, v[e]);
    } else if constexpr (DT == I8_F32) {
        struct __attribute__((packed, aligned(4))) V { float f[8]; } u;
#pragma unroll
        for (int e = 0; e < 8; e++) u.f[e] = v[e];
        *reinterpret_cast<V *>(static_cast<float *>(row) + i) = u;
    } else {
        typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
        u32x4a2 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = i8_bits16<DT>(v[2 * e]) | i8_bits16<DT>(v[2 * e + 1]) << 16;
        *reinterpret_cast<u32x4a2 *>(static_cast<uint16_t *>(row) + i) = w;
    }
}

// The scale of a row whose largest magnitude is amax, never below the smallest normal number; NaN
// where a value is not finite (amax is then infinite or NaN).
__device__ __forceinline__ float i8_scale(float amax) {
    if (!(amax < INFINITY)) return __uint_as_float(0x7fc00000u);
    return amax == 0.f ? 0.f : fmaxf(amax / 127.f, 0x1p-126f);
}
// x / s to the nearest code, ties to even, decided as if the quotient were exact; inv: 1 / s.
// rint of the product is the answer or, next to a tie, one beside it; what is left, x - q s, is
// exact in f32 (a multiple of the operands' last place no larger than about s), so its comparison
// with s / 2 decides.
__device__ __forceinline__ uint32_t i8_code(float x, float s, float inv) {
    const float q = rintf(x * inv), left = fmaf(-q, s, x), most = 0.5f * s;
    const int i = (int)q;
    const bool move = fabsf(left) > most || (fabsf(left) == most && (i & 1));
    return (uint32_t)(move ? left > 0.f ? i + 1 : i - 1 : i) & 0xffu;
}
template <int CTRL>
__device__ __forceinline__ uint32_t i8_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
// the same lanes of a value's words elsewhere in the wave
template <int CTRL, typename V>
__device__ __forceinline__ V i8_dpp_words(V v) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, i8_dpp<CTRL>(__builtin_bit_cast(uint32_t, v)));
    } else {
        const uint64_t w = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(V, (uint64_t)i8_dpp<CTRL>((uint32_t)w) | (uint64_t)i8_dpp<CTRL>((uint32_t)(w >> 32)) << 32);
    }
}
// v of all lanes in every lane: within rows of 16 by DPP, between them by swaps of rows and halves.  Each step joins the
// same two parts in all lanes that hold them, so that a sum rounds alike in every lane (a rotation by 4 joins a quad with the
// one before it in some lanes and the one behind it in others).
template <typename V, typename F>
__device__ __forceinline__ V i8_wave_all(V v, F f) {
    v = f(v, i8_dpp_words<0xB1>(v));   // quad_perm [1,0,3,2]
    v = f(v, i8_dpp_words<0x4E>(v));   // quad_perm [2,3,0,1]
    v = f(v, i8_dpp_words<0x141>(v));  // row_half_mirror
    v = f(v, i8_dpp_words<0x140>(v));  // row_mirror
    auto both = [&](auto swap) {
        if constexpr (sizeof(V) == 4) {
            const auto r = swap(__builtin_bit_cast(uint32_t, v));
            v = f(__builtin_bit_cast(V, (uint32_t)r[0]), __builtin_bit_cast(V, (uint32_t)r[1]));
        } else {
            const uint64_t w = __builtin_bit_cast(uint64_t, v);
            const auto lo = swap((uint32_t)w), hi = swap((uint32_t)(w >> 32));
            v = f(__builtin_bit_cast(V, (uint64_t)(uint32_t)lo[0] | (uint64_t)(uint32_t)hi[0] << 32),
                  __builtin_bit_cast(V, (uint64_t)(uint32_t)lo[1] | (uint64_t)(uint32_t)hi[1] << 32));
        }
    };
    both([](uint32_t u) { return __builtin_amdgcn_permlane16_swap(u, u, false, false); });
    both([](uint32_t u) { return __builtin_amdgcn_permlane32_swap(u, u, false, false); });
    return v;
}
struct I8Sum {
    __device__ double operator()(double a, double b) const { return a + b; }
};
struct I8Max {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};

// magnitudes as the bits of their absolute values: their order is the magnitudes', infinity and NaN
// above all of them
__device__ __forceinline__ uint32_t i8_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ void i8_codes8(const float v[8], float s, float inv, bool live, uint32_t c[2]) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        c[h] = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) c[h] |= i8_code(v[4 * h + e], s, inv) << (8 * e);
        if (!live) c[h] = 0;
    }
}

// An output from the codes' sum: acc s t + b, f32 where the scales' product can neither overflow
// nor lose bits (2^-60 to 2^44 each: what 8-bit codes of any usual values have), else in 64 bits
// and rounded once.  Which of the two goes by the value's own scales, so that the same bits come
// out whatever kernel forms it.
__device__ __forceinline__ bool i8_usual(float scale) { return scale >= 0x1p-60f && scale <= 0x1p44f; }
__device__ __forceinline__ float i8_result(int acc, float s, float t, float b) { return fmaf((float)acc, s * t, b); }
__device__ __forceinline__ float i8_result_wide(int acc, float s, float t, float b) {
    return i8_usual(s) && i8_usual(t) ? i8_result(acc, s, t, b) : (float)((double)acc * (double)s * (double)t + (double)b);
}
// g / (1 + exp(-g)) u, for an output of type OUT.  F32: exp as 2^(h + l) with h + l = -g log2(e) to 48 bits, where a
// plain product would be off by |g| 2^-24 of the result; what l adds is kept beside 1, so that an h beyond the
// exponent's range leaves no inf - inf.  FAR: gates below I8_FAR take 1 + exp(-g) and g by 2^-64, and neither the sum nor
// its reciprocal, which is never subnormal, leaves the range before g / (1 + exp(-g)) itself is below f32's least value.
// Others have the same bits with and without.
constexpr float I8_FAR = -80.f;
template <int OUT, bool FAR = true>
__device__ __forceinline__ float i8_silu_mul(float g, float u) {
    constexpr float L = 1.44269502f, LO = 1.92596303e-8f, LN2 = 0.693147182f;  // log2(e), and what L leaves of it
    const float h = i8_f32(-g * L);  // (as rounded: what the rounding left is l's)
    const bool far = FAR && g < I8_FAR;
    const float one = far ? 0x1p-64f : 1.f, e = __builtin_amdgcn_exp2f(far ? h - 64.f : h);
    float d;
    if constexpr (OUT == I8_F32) {
        const float l = fmaf(-g, LO * LN2, fmaf(fmaf(-g, L, -h), LN2, 1.f));
        d = fmaf(e, __builtin_amdgcn_fmed3f(l, 0.9f, 1.1f), one);
    } else {
        d = one + e;
    }
    return g * one * __builtin_amdgcn_rcpf(d) * u;
}
#endif

}  // namespace lbq
