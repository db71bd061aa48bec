// lbq_i8_gemm.hip -- products of 8-bit codes by tiles, scales and biases in the epilogue.
#include "lbq_i8.hpp"

#include "lbq_internal.hpp"

namespace lbq {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

// a buffer resource over [p, p + bytes), wave-uniform; reads past it give zero
__device__ __forceinline__ __amdgpu_buffer_rsrc_t i8_rsrc(const void *p, int64_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) |
                       ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) << 32);
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(u), (short)0, __builtin_amdgcn_readfirstlane((int)bytes),
                                             0x00020000);
}

struct I8Grid {
    int tiles_m, tiles_n;      // tiles_n: of all weights
    int tile_end[I8_GROUP];  // the first column tile behind each weight's
};

// y = s (A B^T) t + b for a tile of BM tokens by BN channels, A the tokens' codes and B the weight's.
// Both come to LDS by loads that pass the registers by, a stage of 128 bytes of each row at a time into two
// buffers: stage s + 2 is asked for as soon as every wave has its last operands of stage s.  A row's eight
// 16-byte pieces are permuted by (row / 2) & 7, so that the 16 lanes that read at once fall on different
// banks.  A wave has TM x TN tiles of 32 x 32, its operands of the next 32 bytes of k read under this
// one's products.  PAIR: every other 32 channels of a tile are the second weight's, so that a wave holds
// both factors of its outputs.
template <int WM, int WN, int TM, int TN, bool PAIR, int OUT>
__global__ __launch_bounds__(64 * WM * WN) void k_i8_gemm(I8Linear a, I8Grid g) {
    constexpr int NW = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN, BO = PAIR ? BN / 2 : BN;
    constexpr int RA = BM / 8 / NW, RB = BN / 8 / NW;  // staging instructions per wave
    static_assert(RA * 8 * NW == BM && RB * 8 * NW == BN && NW % 2 == 0 && (!PAIR || TN % 2 == 0), "whole staging instructions per wave");
    __shared__ __align__(1024) uint8_t As0[BM * 128], As1[BM * 128];
    __shared__ __align__(1024) uint8_t Bs0[BN * 128], Bs1[BN * 128];
    // neighbouring tiles on one XCD
    const int G = (int)gridDim.x, L = (int)blockIdx.x, X = L & 7;
    const int T = X * (G >> 3) + min(X, G & 7) + (L >> 3);
    const int tm = T % g.tiles_m;
    int tn = T / g.tiles_m, wi = 0;
    if constexpr (!PAIR) {
        while (wi < I8_GROUP - 1 && tn >= g.tile_end[wi]) wi++;
        if (wi) tn -= g.tile_end[wi - 1];
    }
    const int64_t kp = a.kp, m0 = (int64_t)tm * BM;
    const int N = a.n[wi], n0 = tn * BO, ns = (int)(kp / 128);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, lr = lane & 31;
    const int wm = wave / WN, wn = wave % WN;

    const __amdgpu_buffer_rsrc_t ar = i8_rsrc(a.codes + m0 * kp, (a.m - m0 < BM ? a.m - m0 : BM) * kp);
    const int64_t brows = N - n0 < BO ? N - n0 : BO;
    const __amdgpu_buffer_rsrc_t br = i8_rsrc(a.w[wi] + n0 * kp, brows * kp);
    const __amdgpu_buffer_rsrc_t ur = i8_rsrc(a.w[PAIR ? 1 : wi] + n0 * kp, brows * kp);
    // lane l of an instruction fills row l / 8, piece l % 8 of its 8 rows; the rows' number / 8 has
    // the wave's parity (NW is even)
    const int ch = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
    const uint32_t v = (uint32_t)((lane >> 3) * (int)kp + 16 * ch);
    // stage s into buffer `buf`; past the last, zeros (no memory access).  Straight-line code with the
    // buffers' names in it: a load to LDS that the compiler cannot tell from a read's buffer makes it wait
    // for the load before the read.
    auto stage_in = [&](int s, int buf) __attribute__((always_inline)) {
        const uint32_t v0 = s < ns ? v : 0x80000000u;
        const int k0 = s * 128;
#pragma unroll
        for (int j = 0; j < RA; j++) {
            const int rb = wave + NW * j;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ar, (__attribute__((address_space(3))) void *)((buf ? As1 : As0) + 1024 * rb), 16, v0,
                                                     8 * rb * (int)kp + k0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < RB; j++) {
            const int rb = wave + NW * j;
            // (PAIR: rows 64 f .. 64 f + 31 are the first weight's 32 f and on, the next 32 the second's)
            const int row = PAIR ? 32 * (rb >> 3) + 8 * (rb & 3) : 8 * rb;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(PAIR && (rb >> 2 & 1) ? ur : br,
                                                     (__attribute__((address_space(3))) void *)((buf ? Bs1 : Bs0) + 1024 * rb), 16, v0,
                                                     row * (int)kp + k0, 0, 0);
        }
    };
    // byte offsets of a lane's operands of k-step ks, kept as plain numbers (a chain of pointer steps hides
    // from the compiler which buffer it points into)
    int oa[4], ob[4];
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
        const int o = lr * 128 + 16 * ((2 * ks + h) ^ ((lr >> 1) & 7));
        oa[ks] = o + wm * TM * 4096;
        ob[ks] = o + wn * TN * 4096;
        asm volatile("" : "+v"(oa[ks]), "+v"(ob[ks]));
    }
    intx16 acc[TM][TN] = {};
    intx4 xa[2][TM], xb[2][TN];  // operands of this k-step and the next
    auto read = [&](int buf, int ks, int r, int q) __attribute__((always_inline)) {
        if (q < TN) xb[r][q] = *reinterpret_cast<const intx4 *>((buf ? Bs1 : Bs0) + (ob[ks] + q * 4096));
        else xa[r][q - TN] = *reinterpret_cast<const intx4 *>((buf ? As1 : As0) + (oa[ks] + (q - TN) * 4096));
    };
    // the products of the k-step in xa[r], xb[r], each followed by its share of the next one's reads
    auto step = [&](int r, int buf, int ks) __attribute__((always_inline)) {
        constexpr int NM = TM * TN, NR = TM + TN, H = NM > NR ? NM / 2 : NM;
#pragma unroll
        for (int u = 0; u < NM; u++) {
            const int j = u % TN, i = u / TN;
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa[r][i], xb[r][j], acc[i][j], 0, 0, 0);
            if (u < H) {
#pragma unroll
                for (int q = u * NR / H; q < (u + 1) * NR / H; q++) read(buf, ks, r ^ 1, q);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    stage_in(0, 0);
    stage_in(1, 1);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < TN + TM; q++) read(0, 0, 0, q);
    auto stage = [&](int s, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < 3; ks++) step(ks & 1, buf, ks + 1);
        __builtin_amdgcn_s_waitcnt(0);  // this wave's operands, and its loads of stage s + 1
        __syncthreads();
        stage_in(s + 2, buf);
        __builtin_amdgcn_sched_barrier(0);
        step(1, buf ^ 1, 0);
    };
    for (int s = 0; s < ns; s += 2) {  // an odd count ends with a stage of zeros
        stage(s, 0);
        stage(s + 1, 1);
    }
    __builtin_amdgcn_s_waitcnt(0);  // the loads past the last stage

    // lane: channel lr of a 32 x 32 tile, its tokens 8 (v / 4) + 4 h + v % 4
    constexpr int NJ = PAIR ? TN / 2 : TN;
    float tc[TN], bc[TN];
    bool usual = true;
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int wj = PAIR ? j & 1 : wi, n = n0 + 32 * (PAIR ? (wn * TN + j) / 2 : wn * TN + j) + lr;
        tc[j] = n < N ? a.t[wj][n] : 1.f;
        bc[j] = n < N && a.bias[wj] ? a.bias[wj][n] : 0.f;
        usual &= i8_usual(tc[j]);
    }
    void *y = a.y[PAIR ? 0 : wi];
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t mt = m0 + 32 * (wm * TM + i) + 4 * h;
        if (mt - 4 * h >= a.m) break;
        float sr[16];
        bool plain = usual;
#pragma unroll
        for (int v = 0; v < 16; v++) {
            const int64_t m = mt + 8 * (v >> 2) + (v & 3);
            sr[v] = m < a.m ? a.scales[m] : 1.f;
            plain &= i8_usual(sr[v]);
        }
        auto out = [&](auto result) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int n = n0 + 32 * (wn * NJ + j) + lr;
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int64_t m = mt + 8 * (v >> 2) + (v & 3);
                    float o;
                    if constexpr (PAIR)
                        o = i8_silu_mul(result(acc[i][2 * j][v], sr[v], tc[2 * j], bc[2 * j]),
                                        result(acc[i][2 * j + 1][v], sr[v], tc[2 * j + 1], bc[2 * j + 1]));
                    else o = result(acc[i][j][v], sr[v], tc[j], bc[j]);
                    if (m < a.m && n < N) i8_store<OUT>(y, m * N + n, o);
                }
            }
        };
        // (one branch a wave, not a choice a value)
        if (__all(plain)) out([](int c, float s, float t, float b) { return i8_result(c, s, t, b); });
        else out([](int c, float s, float t, float b) { return i8_result_wide(c, s, t, b); });
    }
}

template <int WM, int WN, int TM, int TN, bool PAIR>
hipError_t run(const I8Linear &a, hipStream_t st) {
    constexpr int BM = 32 * WM * TM, BO = 32 * WN * TN / (PAIR ? 2 : 1);
    I8Grid g = {(int)((a.m + BM - 1) / BM), 0, {}};
    for (int i = 0; i < I8_GROUP; i++) {
        if (i < (PAIR ? 1 : a.count)) g.tiles_n += (a.n[i] + BO - 1) / BO;
        g.tile_end[i] = g.tiles_n;
    }
    const unsigned blocks = (unsigned)((int64_t)g.tiles_m * g.tiles_n);
    if (a.out == I8_F32) k_i8_gemm<WM, WN, TM, TN, PAIR, I8_F32><<<blocks, 64 * WM * WN, 0, st>>>(a, g);
    else if (a.out == I8_F16) k_i8_gemm<WM, WN, TM, TN, PAIR, I8_F16><<<blocks, 64 * WM * WN, 0, st>>>(a, g);
    else k_i8_gemm<WM, WN, TM, TN, PAIR, I8_BF16><<<blocks, 64 * WM * WN, 0, st>>>(a, g);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_i8_linear(const I8Linear &a, hipStream_t st) {
    return a.pair ? run<2, 2, 2, 2, true>(a, st) : run<2, 2, 2, 2, false>(a, st);
}

}  // namespace lbq
