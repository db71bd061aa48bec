// lbq_i8_gemm.hip -- products of 8-bit codes by tiles, scales and biases in the epilogue.
#include "lbq_i8.hpp"

#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "lbq_internal.hpp"

namespace lbq {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint64_t uniform64(const void *p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) |
           ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) << 32);
}
// a buffer resource over [p, p + bytes), wave-uniform: reads past it give zero, writes nothing
__device__ __forceinline__ intx4 i8_rsrc(const void *p, int64_t bytes) {
    const uint64_t a = uniform64(p);
    return {(int)(uint32_t)a, (int)(uint32_t)(a >> 32) & 0xffff, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
// 16 or 4 bytes a lane from rsrc + v + s to LDS at `to` + 16 or 4 lane, past the registers.  Written out, since the
// compiler would wait for all such loads before a read of LDS that it cannot tell from their targets; who reads
// what they bring waits for vmcnt, which counts them in order.
__device__ __forceinline__ void i8_load_lds(intx4 rsrc, uint32_t to, uint32_t v, int s) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(v), "s"(rsrc), "s"(s) : "memory");
}
__device__ __forceinline__ void i8_load_lds4(intx4 rsrc, uint32_t to, uint32_t v) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(v), "s"(rsrc) : "memory");
}
// all but the last N of the wave's loads are there, and all its reads of LDS
template <int N>
__device__ __forceinline__ void i8_wait() {
    static_assert(N < 64, "vmcnt has six bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void i8_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// two values as 16-bit ones, rounded to nearest even, the first in the low half
template <int OUT>
__device__ __forceinline__ uint32_t i8_pack(float a, float b) {
    if constexpr (OUT == I8_F16) {
        typedef _Float16 half2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, half2{(_Float16)i8_f32(a), (_Float16)i8_f32(b)});
    } else {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, bf2{(__bf16)a, (__bf16)b});
    }
}

// A tile's shape: WM x WN waves of TM x TN tiles of 32 x 32, D stages of 128 bytes of each row in LDS.  PAIR: every
// other 32 of the BN channels are the second weight's, BO outputs a row.
template <int WM_, int WN_, int TM_, int TN_, int D_, bool PAIR_>
struct Tile {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, D = D_;
    static constexpr bool PAIR = PAIR_;
    static constexpr int NW = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN, BO = PAIR ? BN / 2 : BN;
    static constexpr int RA = BM / 8 / NW, RB = BN / 8 / NW, RL = RA + RB;  // loads per wave and stage
    static_assert(RA * 8 * NW == BM && RB * 8 * NW == BN && NW % 2 == 0 && (!PAIR || TN % 2 == 0), "whole loads per wave");
    static_assert(TM * TN > 2 || D % 2 == 0, "two register sets of a stage's operands");
    // behind the stages, scales of tokens and channels and biases in pieces of 64
    static constexpr int STAGE = (BM + BN) * 128, PM = (BM + 63) / 64, PN = (BN + 63) / 64, VECTORS = PM + 2 * PN;
    static constexpr int LDS = D * STAGE + 256 * VECTORS;
};

// y = s (A B^T) t + b for the tile at token m0 and channel n0 of weight wi (PAIR: of both), A the tokens' codes and
// B the weight's.  Both come to LDS by loads that pass the registers by; stage s + D is asked for as soon as
// every wave has its last operands of stage s.  A row's eight 16-byte pieces are permuted by (row / 2) & 7, so that
// the 16 lanes that read at once fall on different banks.  Where a k-step of 32 has more than two products a
// wave, the next one's operands are read under them, and the loads go out one behind each; where it has fewer, a
// whole stage's operands are read ahead.
// 4096 x 14336 -> 4096 188 us, 2.55 POP/s; 2048 tokens, gate and up of 14336 x 4096 216 us, 2.23.  Bound by the card's power: the
// matrix pipes are busy 55 to 70 % of cycles at 1.8 GHz, and on codes of zeros, which take less of it, the rate is 3.0.  512 tokens over
// 6144 channels of 4096 (192 tiles of 128 x 128, a call on codes made before) 19.0 us, 22.4 where the weights come out of memory: 5.4 of
// a launch's start and end, and 0.40 or 0.52 a stage, of which the matrix instructions are 0.21; over k of 512 to 8192 alike, so that it is
// not the lines missing in an L2.  All CUs take in 16 TB/s together there (256 tiles of 128 x 64: 20 to 25).  Stages of 64 bytes in 3 to 5 slots took 214 to 228 us
// for 190 to 199, four waves of 128 x 128 each 307 (registers spill).
template <class T, int OUT>
__device__ __forceinline__ void i8_tile(const I8Linear &a, int64_t m0, int n0, int wi, uint8_t *lds_base) {
    constexpr int TM = T::TM, TN = T::TN, D = T::D, NW = T::NW, RA = T::RA, RL = T::RL, BM = T::BM, BO = T::BO;
    constexpr bool PAIR = T::PAIR;
    const int64_t kp = a.kp;
    const int N = a.n[wi], ns = (int)(kp / 128);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, lr = lane & 31;
    const int wm = wave / T::WN, wn = wave % T::WN;

    const int64_t rows = a.m - m0 < BM ? a.m - m0 : BM, cols = N - n0 < BO ? N - n0 : BO;
    const intx4 ar = i8_rsrc(a.codes + m0 * kp, rows * kp);
    const intx4 br = i8_rsrc(a.w[wi] + n0 * kp, cols * kp), ur = i8_rsrc(a.w[PAIR ? 1 : wi] + n0 * kp, cols * kp);
    // lane l of an instruction fills row l / 8, piece l % 8 of its 8 rows; the rows' number / 8 has
    // the wave's parity (NW is even)
    const int ch = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
    const uint32_t v = (uint32_t)((lane >> 3) * (int)kp + 16 * ch);
    const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds_base);
    // load q of stage s into slot b; past the last stage, zeros (no memory access)
    auto load = [&](int s, int b, int q) __attribute__((always_inline)) {
        const uint32_t v0 = s < ns ? v : 0x80000000u, to = lds + b * T::STAGE;
        if (q < RA) {
            const int rb = wave + NW * q;
            i8_load_lds(ar, to + 1024 * rb, v0, 8 * rb * (int)kp + s * 128);
        } else {
            const int rb = wave + NW * (q - RA);
            // (PAIR: rows 64 f .. 64 f + 31 are the first weight's 32 f and on, the next 32 the second's)
            const int row = PAIR ? 32 * (rb >> 3) + 8 * (rb & 3) : 8 * rb;
            i8_load_lds(PAIR && (rb >> 2 & 1) ? ur : br, to + BM * 128 + 1024 * rb, v0, row * (int)kp + s * 128);
        }
    };
    // scales and biases, before the stages: the first wait of any stage covers them.  Channels' lie in the
    // tile's order (PAIR: the first weight's BO, then the second's)
    float *vec = reinterpret_cast<float *>(lds_base + D * T::STAGE);
    for (int q = wave; q < T::VECTORS; q += NW) {
        const uint32_t to = lds + D * T::STAGE + 256 * q;
        if (q < T::PM) {
            i8_load_lds4(i8_rsrc(a.scales + m0, rows * 4), to, 256 * q + 4 * lane);
        } else {
            const bool bias = q >= T::PM + T::PN;
            const int c = 64 * (q - T::PM - (bias ? T::PN : 0)), w = PAIR && c >= BO ? 1 : wi;  // (BO is a multiple of 64 where PAIR)
            const float *p = bias ? a.bias[w] : a.t[w];
            if (p) i8_load_lds4(i8_rsrc(p + n0, cols * 4), to, 4 * (c - (PAIR && c >= BO ? BO : 0) + lane));
        }
    }
    static_assert(!PAIR || BO % 64 == 0, "pieces of one weight");

    // byte offsets of a lane's operands of k-step ks
    int oa[4], ob[4];
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
        const int o = lr * 128 + 16 * ((2 * ks + h) ^ ((lr >> 1) & 7));
        oa[ks] = o + wm * TM * 4096;
        ob[ks] = o + wn * TN * 4096 + BM * 128;
        asm volatile("" : "+v"(oa[ks]), "+v"(ob[ks]));
    }
    intx16 acc[TM][TN] = {};
#pragma unroll
    for (int s = 0; s < D; s++)
#pragma unroll
        for (int q = 0; q < RL; q++) load(s, s, q);
    i8_wait<(D - 1) * RL>();
    i8_barrier();
    if constexpr (TM * TN > 2) {
        intx4 xa[2][TM], xb[2][TN];  // operands of this k-step and the next
        auto read = [&](int b, int ks, int r, int q) __attribute__((always_inline)) {
            if (q < TN) xb[r][q] = *reinterpret_cast<const intx4 *>(lds_base + b * T::STAGE + (ob[ks] + q * 4096));
            else xa[r][q - TN] = *reinterpret_cast<const intx4 *>(lds_base + b * T::STAGE + (oa[ks] + (q - TN) * 4096));
        };
        // the products of the k-step in xa[r], xb[r], each followed by its share of the next one's reads (slot b,
        // k-step ks) and, where ls >= 0, of the loads of stage ls into slot lb
        auto step = [&](int r, int b, int ks, int ls, int lb) __attribute__((always_inline)) {
            constexpr int NM = TM * TN, NR = TM + TN, H = NM > NR ? NM / 2 : NM;
#pragma unroll
            for (int u = 0; u < NM; u++) {
                const int j = u % TN, i = u / TN;
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa[r][i], xb[r][j], acc[i][j], 0, 0, 0);
                if (u < H) {
#pragma unroll
                    for (int q = u * NR / H; q < (u + 1) * NR / H; q++) read(b, ks, r ^ 1, q);
                }
                if (ls >= 0) {
#pragma unroll
                    for (int q = u * RL / NM; q < (u + 1) * RL / NM; q++) load(ls, lb, q);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
#pragma unroll
        for (int q = 0; q < TN + TM; q++) read(0, 0, 0, q);
        for (int s = 0; s < ns; s += D) {
#pragma unroll
            for (int i = 0; i < D; i++) {
                if (i && s + i >= ns) break;
#pragma unroll
                for (int ks = 0; ks < 3; ks++) step(ks & 1, i, ks + 1, -1, 0);
                i8_wait<(D - 2) * RL>();  // this wave's operands, and its loads of stage s + i + 1
                i8_barrier();
                step(1, (i + 1) % D, 0, s + i + D, i);
            }
        }
    } else {
        intx4 xa[2][4][TM], xb[2][4][TN];
        auto read = [&](int b, int r) __attribute__((always_inline)) {
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
#pragma unroll
                for (int q = 0; q < TN; q++) xb[r][ks][q] = *reinterpret_cast<const intx4 *>(lds_base + b * T::STAGE + (ob[ks] + q * 4096));
#pragma unroll
                for (int q = 0; q < TM; q++) xa[r][ks][q] = *reinterpret_cast<const intx4 *>(lds_base + b * T::STAGE + (oa[ks] + q * 4096));
            }
        };
        read(0, 0);
        for (int s = 0; s < ns; s += D) {
#pragma unroll
            for (int i = 0; i < D; i++) {
                if (i && s + i >= ns) break;
                i8_wait<(D - 2) * RL>();  // this wave's operands, and its loads of stage s + i + 1
                i8_barrier();
                read((i + 1) % D, (i + 1) & 1);
#pragma unroll
                for (int q = 0; q < RL; q++) load(s + i + D, i, q);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
#pragma unroll
                    for (int u = 0; u < TM * TN; u++)
                        acc[u / TN][u % TN] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa[i & 1][ks][u / TN], xb[i & 1][ks][u % TN], acc[u / TN][u % TN], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    i8_wait<0>();  // the loads past the last stage

    // lane: channel lr of a 32 x 32 tile, its tokens 8 (v / 4) + 4 h + v % 4
    constexpr int NJ = PAIR ? TN / 2 : TN;
    float tc[TN], bc[TN];
    bool usual = true;
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int c = PAIR ? 32 * ((wn * TN + j) / 2) + lr + (j & 1 ? BO : 0) : 32 * (wn * TN + j) + lr;
        const bool live = n0 + c - (PAIR && j & 1 ? BO : 0) < N;
        tc[j] = vec[64 * T::PM + c];
        bc[j] = a.bias[PAIR ? j & 1 : wi] ? vec[64 * (T::PM + T::PN) + c] : 0.f;
        usual &= !live || i8_usual(tc[j]);
    }
    for (int i = lane; i < 32 * TM; i += 64) usual &= 32 * TM * wm + i >= rows || i8_usual(vec[32 * TM * wm + i]);
    char *y = static_cast<char *>(a.y[PAIR ? 0 : wi]);
    constexpr int SIZE = OUT == I8_F32 ? 4 : 2;
    // (16-bit outputs of two neighbouring channels in one store, where a row's are 4-byte aligned: an even lane
    // stores its and its neighbour's of token e, an odd one of token e + 1)
    const bool even = OUT != I8_F32 && N % 2 == 0 && (reinterpret_cast<uintptr_t>(y) & 3) == 0;
    const uint32_t mix = lane & 1 ? 0x03020706u : 0x05040100u;
    auto out = [&](auto result, auto wide) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int64_t mt = m0 + 32 * (wm * TM + i);
            if (mt >= a.m) break;
            floatx4 sr[4];
#pragma unroll
            for (int q = 0; q < 4; q++) sr[q] = *reinterpret_cast<const floatx4 *>(vec + 32 * (wm * TM + i) + 8 * q + 4 * h);
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int n = n0 + 32 * (wn * NJ + j) + lr;
                uint32_t vo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) vo[e] = n < N ? ((uint32_t)(4 * h + e) * (uint32_t)N + (uint32_t)n) * SIZE : 0x80000000u;
                // (even: e = 0 and 2, from the pair's first channel on and for the lane's token)
                const uint32_t step = even && lane & 1 ? ((uint32_t)N - 1) * SIZE : 0;
                // (the pair's outputs.  One question for a lane's 16 gates: asked of each, 2048 x 512 -> 14336 takes 51.7 us for 50.0)
                float both[16];
                if constexpr (PAIR) {
                    float g[16], few[4];
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        g[v] = result(acc[i][2 * j][v], sr[v / 4][v % 4], tc[2 * j], bc[2 * j]);
                        both[v] = result(acc[i][2 * j + 1][v], sr[v / 4][v % 4], tc[2 * j + 1], bc[2 * j + 1]);
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++) few[q] = fminf(fminf(fminf(g[4 * q], g[4 * q + 1]), g[4 * q + 2]), g[4 * q + 3]);
                    const float least = fminf(fminf(fminf(few[0], few[1]), few[2]), few[3]);
                    if (wide || __any(least < I8_FAR)) {
#pragma unroll
                        for (int v = 0; v < 16; v++) both[v] = i8_silu_mul<OUT, true>(g[v], both[v]);
                    } else {
#pragma unroll
                        for (int v = 0; v < 16; v++) both[v] = i8_silu_mul<OUT, false>(g[v], both[v]);
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int left = (int)(a.m - mt < 32 ? a.m - mt : 32) - 8 * q;
                    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                        reinterpret_cast<void *>(uniform64(y + (mt + 8 * q) * N * SIZE)), (short)0,
                        __builtin_amdgcn_readfirstlane((left < 0 ? 0 : left > 8 ? 8 : left) * N * SIZE), 0x00020000);
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (PAIR) o[e] = both[4 * q + e];
                        else o[e] = result(acc[i][j][4 * q + e], sr[q][e], tc[j], bc[j]);
                    }
                    if constexpr (OUT == I8_F32) {
#pragma unroll
                        for (int e = 0; e < 4; e++) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[e]), rs, vo[e], 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const uint32_t own = i8_pack<OUT>(o[e], o[e + 1]);
                            if (even) {
                                const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)own, 0xB1, 0xf, 0xf, true);  // lane ^ 1's
                                __builtin_amdgcn_raw_buffer_store_b32(__builtin_amdgcn_perm(other, own, mix), rs, vo[e] + step, 0, 0);
                            } else {
                                __builtin_amdgcn_raw_buffer_store_b16((uint16_t)own, rs, vo[e], 0, 0);
                                __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(own >> 16), rs, vo[e + 1], 0, 0);
                            }
                        }
                    }
                }
            }
        }
    };
    // (one branch a wave, not a choice a value; the wide form, hardly ever taken, asks for no far gates)
    if (__all(usual)) out([](int c, float s, float t, float b) { return i8_result(c, s, t, b); }, std::false_type{});
    else out([](int c, float s, float t, float b) { return i8_result_wide(c, s, t, b); }, std::true_type{});
}

// Tiles of shape T over the column tiles of each weight, the last columns, from tile `wide` on, by tiles of shape U
// with as many channels and fewer tokens: what is left of a last round over the CUs.  Tiles run down bands of
// I8_BAND row tiles, neighbours on one XCD: the 32 tiles that an XCD works on at once share four panels of A and
// eight of B.
struct I8Grid {
    int tiles_n, wide, rows_t, rows_u;  // column tiles in all and of shape T, row tiles of each shape
    int tile_end[I8_GROUP];             // the first column tile behind each weight's
};
constexpr int I8_BAND = 4;

template <class T, class U, int OUT>
__global__ __launch_bounds__(64 * T::NW) void k_i8_gemm(I8Linear a, I8Grid g) {
    static_assert(T::NW == U::NW && T::BO == U::BO, "one launch shape");
    __shared__ __align__(1024) uint8_t lds[T::LDS > U::LDS ? T::LDS : U::LDS];
    const int first = g.wide * g.rows_t;
    int L = (int)blockIdx.x, G = first, columns = g.wide, rows = g.rows_t, from = 0;
    if (L >= first) L -= first, G = (int)gridDim.x - first, columns = g.tiles_n - g.wide, rows = g.rows_u, from = g.wide;
    const int X = L & 7, at = X * (G >> 3) + min(X, G & 7) + (L >> 3);
    const int band = at / (I8_BAND * columns), in = at - band * I8_BAND * columns, deep = min(I8_BAND, rows - band * I8_BAND);
    const int tm = band * I8_BAND + in % deep;
    int tn = from + in / deep, wi = 0;
    if constexpr (!T::PAIR) {
        while (wi < I8_GROUP - 1 && tn >= g.tile_end[wi]) wi++;
        if (wi) tn -= g.tile_end[wi - 1];
    }
    if constexpr (T::BM == U::BM) {
        i8_tile<T, OUT>(a, (int64_t)tm * T::BM, tn * T::BO, wi, lds);
    } else {
        if ((int)blockIdx.x < first) i8_tile<T, OUT>(a, (int64_t)tm * T::BM, tn * T::BO, wi, lds);
        else i8_tile<U, OUT>(a, (int64_t)tm * U::BM, tn * U::BO, wi, lds);
    }
}

template <class T>
int columns(const I8Linear &a, int *end) {
    int n = 0;
    for (int i = 0; i < I8_GROUP; i++) {
        if (i < (T::PAIR ? 1 : a.count)) n += (a.n[i] + T::BO - 1) / T::BO;
        end[i] = n;
    }
    return n;
}

// the columns from tile `wide` on by shape U
template <class T, class U>
hipError_t run(const I8Linear &a, int wide, hipStream_t st) {
    I8Grid g = {};
    g.tiles_n = columns<T>(a, g.tile_end);
    g.wide = std::min(wide, g.tiles_n);
    g.rows_t = (int)((a.m + T::BM - 1) / T::BM), g.rows_u = (int)((a.m + U::BM - 1) / U::BM);
    const unsigned blocks = (unsigned)((int64_t)g.wide * g.rows_t + (int64_t)(g.tiles_n - g.wide) * g.rows_u);
    if (a.out == I8_F32) k_i8_gemm<T, U, I8_F32><<<blocks, 64 * T::NW, 0, st>>>(a, g);
    else if (a.out == I8_F16) k_i8_gemm<T, U, I8_F16><<<blocks, 64 * T::NW, 0, st>>>(a, g);
    else k_i8_gemm<T, U, I8_BF16><<<blocks, 64 * T::NW, 0, st>>>(a, g);
    return hipGetLastError();
}

// A stage's time goes by what is taken in, the rows and channels of a tile, so that large tiles pay only where they fill the
// CUs.  us of the first round of tiles, one a CU, and of each further one at k = 4096 (measured, weights out of memory; other k by
// their length alike).
template <class T>
float cost(const I8Linear &a, float first, float next) {
    int end[I8_GROUP];
    const int64_t tiles = (int64_t)columns<T>(a, end) * ((a.m + T::BM - 1) / T::BM);
    return first + next * (float)((tiles + num_cus() - 1) / num_cus() - 1);
}
template <bool PAIR>
hipError_t tiles(const I8Linear &a, hipStream_t st) {
    using Big = Tile<2, 4, 4, 2, 2, PAIR>;     // 256 x 256
    using Half = Tile<2, 4, 2, 2, 3, PAIR>;    // 128 x 256
    // 128 x 128 (waves of 64 x 32 where a pair does not need two columns: 512 x 4096 -> 6144 a call on codes made before 22.2 to
    // 22.6 us, weights out of memory, for 23.8 of 32 x 64)
    using Square = std::conditional_t<PAIR, Tile<4, 2, 1, 2, 4, true>, Tile<2, 4, 2, 1, 4, false>>;
    using Tall = std::conditional_t<PAIR, Square, Tile<4, 2, 1, 1, 4, false>>;                         // 128 x 64
    using Small = std::conditional_t<PAIR, Tile<2, 2, 1, 2, 4, true>, Tile<2, 2, 1, 1, 4, false>>;     // 64 x 128 or 64 x 64
    using Least = std::conditional_t<PAIR, Small, Tile<1, 2, 1, 1, 6, false>>;                         // 32 x 64
    int end[I8_GROUP];
    // the big tiles' last round, where it is at most half of one, by halves of them
    const int cus = num_cus(), cols = columns<Big>(a, end), rows = (int)((a.m + 255) / 256), rounds = (int)((int64_t)cols * rows / cus);
    const int wide = (int)std::min<int64_t>(cols, (int64_t)rounds * cus / rows);
    const int64_t rest = (int64_t)(cols - wide) * ((a.m + 127) / 128);
    const float big = cost<Big>(a, 58.f, 58.f), mixed = 58.f * rounds + 35.f * (float)((rest + cus - 1) / cus);
    const float half = cost<Half>(a, 33.f, 35.f), square = cost<Square>(a, 22.3f, 22.3f);
    const float tall = PAIR ? square : cost<Tall>(a, 14.7f, 14.7f);
    const float small = PAIR ? cost<Small>(a, 16.f, 15.7f) : cost<Small>(a, 11.5f, 7.2f), least = PAIR ? small : cost<Least>(a, 9.5f, 5.4f);
    const float best = std::min({big, mixed, half, square, tall, small, least});
    if (least == best) return run<Least, Least>(a, INT_MAX, st);
    if (small == best) return run<Small, Small>(a, INT_MAX, st);
    if (tall == best) return run<Tall, Tall>(a, INT_MAX, st);
    if (square == best) return run<Square, Square>(a, INT_MAX, st);
    if (half == best) return run<Half, Half>(a, INT_MAX, st);
    return run<Big, Half>(a, big == best ? INT_MAX : wide, st);
}

}  // namespace

hipError_t launch_i8_linear(const I8Linear &a, hipStream_t st) {
    if (i8_streams(a)) return launch_i8_stream(a, st);
    return a.pair ? tiles<true>(a, st) : tiles<false>(a, st);
}

}  // namespace lbq
