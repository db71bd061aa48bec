// lbq_i8_gemv.hip -- products of 8-bit codes for up to 32 tokens: the weights stream from memory to registers.
#include "lbq_i8.hpp"

#include <algorithm>

#include "lbq_internal.hpp"

namespace lbq {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));

struct I8Stream {
    int ks;                  // waves that share a tile's k: 1, 2, 4 or 8
    int tile_end[I8_GROUP];  // the first tile behind each weight's
};
constexpr int I8_WAVES = 8, I8_LDS = I8_FUSED_CODES + 16 * I8_FUSED_ROWS;

// y = s (A B^T) t + b for up to MT x 16 tokens (A) by tiles of R x 16 channels (B).  A wave holds a tile, or, ks > 1,
// the tile's share of k, and reads both operands as the matrix cores take them, 16 bytes of 16 rows a
// lane: 128 bytes of each row a block, U blocks at once into one of two register sets while the
// other's are multiplied.  Bound by memory: each weight is read once by one wave; the tokens come out of the
// L2, or (FUSED: values quantised by the workgroup, codes and scales as the other kernel's) out of LDS.  Shares
// of k meet in LDS; whole numbers, so that their order does not matter.
// 8 tokens over 128256 channels of 4096 93 us, 5.7 TB/s; 16 tokens, gate and up of 14336 25 us, 4.7 TB/s; one token over 6144 8.5 us,
// of which about 3 are the launch, its values' quantisation and the join.
template <int MT, int R, int U, bool PAIR, bool FUSED, int DX, int OUT>
__global__ __launch_bounds__(64 * I8_WAVES) void k_i8_gemv(I8Linear a, I8Stream g) {
    constexpr int NB = R * (PAIR ? 2 : 1), NV = MT * NB;
    __shared__ __align__(16) int sums[I8_WAVES][NV][64][4];
    __shared__ __align__(16) int8_t xs[FUSED ? I8_LDS : 16];
    __shared__ float sx[FUSED ? I8_FUSED_ROWS : 1];
    __shared__ uint32_t part[I8_WAVES];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), lr = lane & 15, lg = lane >> 4;
    const int per = I8_WAVES / g.ks, share = wave % g.ks;
    const int all = g.tile_end[I8_GROUP - 1], at = (int)blockIdx.x * per + wave / g.ks;
    int tile = min(at, all - 1), wi = 0;  // (waves without a tile repeat the last one, and write nothing)
    if constexpr (!PAIR) {
        while (wi < I8_GROUP - 1 && tile >= g.tile_end[wi]) wi++;
        if (wi) tile -= g.tile_end[wi - 1];
    }
    const int64_t kp = a.kp;
    const int N = a.n[wi], n0 = tile * 16 * R, m = (int)a.m;
    const int blocks = a.kp / 128, b0 = blocks * share / g.ks, b1 = blocks * (share + 1) / g.ks, last = max(b1 - 1, 0);

    // the tile's first row, and a lane's offset from it (rows behind the last repeat it)
    const int8_t *w0[NB];
    uint32_t wo[NB], xo[MT];
#pragma unroll
    for (int i = 0; i < NB; i++) {
        w0[i] = a.w[PAIR ? i & 1 : wi] + n0 * kp;
        wo[i] = (uint32_t)(min(16 * (PAIR ? i >> 1 : i) + lr, N - 1 - n0) * a.kp + 16 * lg);
    }
    const int xstep = FUSED ? a.kp + 16 : a.kp;  // FUSED: rows of codes in LDS, on different banks
#pragma unroll
    for (int i = 0; i < MT; i++) xo[i] = (uint32_t)(min(16 * i + lr, m - 1) * xstep + 16 * lg);

    intx4 w[2][U][NB][2], x[2][U][MT][2];
    auto load_w = [&](int r, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) w[r][u][i][h] = *reinterpret_cast<const intx4 *>(w0[i] + 128 * min(b + u, last) + 64 * h + wo[i]);
    };
    auto load_x = [&](int r, int b) __attribute__((always_inline)) {
        if constexpr (!FUSED)
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) x[r][u][i][h] = *reinterpret_cast<const intx4 *>(a.codes + 128 * min(b + u, last) + 64 * h + xo[i]);
    };
    // scales and biases of the outputs, asked for early where that leaves registers for two workgroups a CU
    constexpr bool EARLY = NV < 4;
    float tc[NB], bc[NB], sc[MT][4];
    auto vectors = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int wj = PAIR ? j & 1 : wi, n = min(n0 + 16 * (PAIR ? j >> 1 : j) + lr, N - 1);
            tc[j] = a.t[wj][n];
            bc[j] = a.bias[wj] ? a.bias[wj][n] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int v = 0; v < 4; v++)
                if constexpr (!FUSED) sc[i][v] = a.scales[min(16 * i + 4 * lg + v, m - 1)];
    };
    if constexpr (EARLY) vectors();
    intx4 acc[MT][NB] = {};
    auto multiply = [&](int r, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (b + u >= b1) break;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const intx4 xv = FUSED ? *reinterpret_cast<const intx4 *>(xs + 128 * (b + u) + 64 * h + xo[i]) : x[r][u][i][h];
#pragma unroll
                    for (int j = 0; j < NB; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv, w[r][u][j][h], acc[i][j], 0, 0, 0);
                }
        }
    };

    if constexpr (FUSED) {
        // rows of 512, 256 or 128 threads; x is asked for before the weights, whose loads it would wait for
        const int lanes = 64 * I8_WAVES >> (m > 2 ? 2 : m - 1), row = min(t / lanes, m - 1), tr = t % lanes;
        const int np = (a.kp / 8 + lanes - 1) / lanes;
        constexpr int P = I8_FUSED_CODES / 8 / (64 * I8_WAVES);
        const char *xr = static_cast<const char *>(a.x.p) + row * a.x.stride * (DX == I8_F32 ? 4 : 2);
        float v[P][8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < P; j++)
            if (j < np) i8_load8<DX>(xr, 8 * (tr + j * lanes), a.k, v[j]);
        load_w(0, b0), load_w(1, b0 + U);
#pragma unroll
        for (int j = 0; j < P; j++)
            if (j < np)
#pragma unroll
                for (int e = 0; e < 8; e++) top = max(top, i8_magnitude(v[j][e]));
        top = i8_wave_all(top, I8Max{});
        if (lane == 0) part[wave] = top;
        __syncthreads();
        const int first = t / lanes * (lanes / 64);
        top = part[first];
        for (int i = 1; i < lanes / 64; i++) top = max(top, part[first + i]);
        const float s = i8_scale(__uint_as_float(top)), inv = 1.f / s;
        if (t / lanes < m) {
            if (tr == 0) sx[row] = s;
#pragma unroll
            for (int j = 0; j < P; j++) {
                const int i = 8 * (tr + j * lanes);
                if (j < np && i < kp) {
                    uint32_t c[2];
                    i8_codes8(v[j], s, inv, s > 0.f, c);
                    *reinterpret_cast<uint2 *>(xs + row * xstep + i) = make_uint2(c[0], c[1]);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < 4; v++) sc[0][v] = sx[min(4 * lg + v, m - 1)];
    } else {
        load_x(0, b0), load_w(0, b0), load_x(1, b0 + U), load_w(1, b0 + U);
    }
    int b = b0;
    for (; b + 3 * U < b1; b += 2 * U) {
        multiply(0, b);
        load_x(0, b + 2 * U), load_w(0, b + 2 * U);
        multiply(1, b + U);
        load_x(1, b + 3 * U), load_w(1, b + 3 * U);
    }
    multiply(0, b);
    if (b + 2 * U < b1) {
        load_x(0, b + 2 * U), load_w(0, b + 2 * U);
        multiply(1, b + U);
        multiply(0, b + 2 * U);
    } else {
        multiply(1, b + U);
    }

    if (g.ks > 1) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NB; j++) *reinterpret_cast<intx4 *>(sums[wave][i * NB + j][lane]) = acc[i][j];
        __syncthreads();
    }
    if constexpr (!EARLY) vectors();
    if (at >= all) return;
    // lane: channel lr of a 16 x 16 tile, its tokens 4 lg + v; value (i, j, v) goes to one of the tile's waves
    const int lead = wave - share;
    void *y = a.y[PAIR ? 0 : wi];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < R; j++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                if (((i * R + j) * 4 + v) % g.ks != share) continue;
                const int n = n0 + 16 * j + lr, tok = 16 * i + 4 * lg + v;
                int c[2];
#pragma unroll
                for (int p = 0; p < (PAIR ? 2 : 1); p++) {
                    const int q = PAIR ? 2 * j + p : j;
                    c[p] = acc[i][q][v];
                    if (g.ks > 1) {
                        c[p] = 0;
                        for (int s = 0; s < g.ks; s++) c[p] += sums[lead + s][i * NB + q][lane][v];
                    }
                }
                if (n >= N || tok >= m) continue;
                float o = i8_result_wide(c[0], sc[i][v], tc[PAIR ? 2 * j : j], bc[PAIR ? 2 * j : j]);
                if constexpr (PAIR) o = i8_silu_mul<OUT>(o, i8_result_wide(c[1], sc[i][v], tc[2 * j + 1], bc[2 * j + 1]));
                i8_store<OUT>(y, (int64_t)tok * N + n, o);
            }
}

template <int R>
int tiles16(const I8Linear &a, int *end) {
    int tiles = 0;
    for (int i = 0; i < I8_GROUP; i++) {
        if (i < (a.pair ? 1 : a.count)) tiles += (a.n[i] + 16 * R - 1) / (16 * R);
        end[i] = tiles;
    }
    return tiles;
}

template <int MT, int R, int U, bool PAIR, bool FUSED, int DX>
hipError_t run(const I8Linear &a, hipStream_t st) {
    I8Stream g = {};
    const int tiles = tiles16<R>(a, g.tile_end), blocks = a.kp / 128;
    g.ks = blocks >= 8 ? 8 : blocks >= 4 ? 4 : blocks >= 2 ? 2 : 1;
    // longer shares where that leaves three quarters of the CUs a workgroup or more.  us in eighths and quarters of k = 4096, a
    // pair, 16 tokens: 8192 channels 17.7 and 23.4, 10240 28.1 and 23.8, 12288 (the first to take quarters) 29.0 and 24.7, 14336 32.0
    // and 25.1, 16384 33.9 and 27.0, 20480 44.2 and 46.5, 28672 57.7 and 50.0; k = 8192: 12288 51.5 and 43.4, 16384 52.1 and 50.4.
    // (Single weights 16.0 and 15.5, 128256 channels 92.7 and 96.3.)
    if (PAIR && R == 2 && tiles / 2 >= num_cus() * 3 / 4) g.ks = std::min(g.ks, 4);
    const unsigned groups = (unsigned)((tiles + I8_WAVES / g.ks - 1) / (I8_WAVES / g.ks));
    if (a.out == I8_F32) k_i8_gemv<MT, R, U, PAIR, FUSED, DX, I8_F32><<<groups, 64 * I8_WAVES, 0, st>>>(a, g);
    else if (a.out == I8_F16) k_i8_gemv<MT, R, U, PAIR, FUSED, DX, I8_F16><<<groups, 64 * I8_WAVES, 0, st>>>(a, g);
    else k_i8_gemv<MT, R, U, PAIR, FUSED, DX, I8_BF16><<<groups, 64 * I8_WAVES, 0, st>>>(a, g);
    return hipGetLastError();
}
template <int R, int U, bool PAIR>
hipError_t fused(const I8Linear &a, hipStream_t st) {
    return a.x.dtype == I8_F32 ? run<1, R, U, PAIR, true, I8_F32>(a, st)
         : a.x.dtype == I8_F16 ? run<1, R, U, PAIR, true, I8_F16>(a, st)
                               : run<1, R, U, PAIR, true, I8_BF16>(a, st);
}
template <bool PAIR>
hipError_t stream(const I8Linear &a, hipStream_t st) {
    int end[I8_GROUP];
    // Two tiles of 16 channels a wave where there are more of them than CUs, so that each token operand is used twice.  us at
    // k = 4096, one tile and two: 4096 channels 6.2 and 7.0, 6144 8.6 and 7.9, 14336 (16 tokens) 18.9 and 16.0, 128256 (8 tokens)
    // 102 and 93.  A fused kernel's registers take two blocks at once (6144: 8.9 us for 9.3), a pair's of two tiles do not.
    const bool two = tiles16<1>(a, end) > num_cus();
    if (a.x.p) return two ? fused<2, PAIR ? 1 : 2, PAIR>(a, st) : fused<1, 2, PAIR>(a, st);
    if (a.m > 16) return run<2, 1, 1, PAIR, false, I8_F32>(a, st);
    return two ? run<1, 2, 1, PAIR, false, I8_F32>(a, st) : run<1, 1, 1, PAIR, false, I8_F32>(a, st);
}

}  // namespace

// Every workgroup quantises the tokens for itself, which saves a launch and its gap (1 token, 4096 channels of 4096: 6.6 us a call for
// 10.1) while the CUs' workgroups are all at work at once; over more channels it costs more than it saves (4 tokens, pair
// of 14336: 28.7 us for 27.1; 128256 channels 101 for 91), and so do more tokens (8: 13.6 for 10.1).
bool i8_quantizes_in_kernel(int64_t m, int64_t k, int64_t channels) {
    return m <= I8_FUSED_ROWS && (m > 2 ? 4 : m) * i8_kp(k) <= I8_FUSED_CODES && channels <= I8_FUSED_CHANNELS;
}

// Up to 16 tokens; up to 32 where a tile of 16 channels a CU is enough: us of this kernel and of the tiles' at k = 4096, 32 tokens,
// 2048 channels 8.0 and 8.8, 4096 8.6 and 9.9 (k = 14336: 22.9 and 30.0), 6144 11.9 and 11.9, 14336 20.6 and 16.2.
bool i8_streams(const I8Linear &a) {
    int end[I8_GROUP];
    return a.m <= 16 || (a.m <= 32 && tiles16<1>(a, end) <= num_cus());
}
hipError_t launch_i8_stream(const I8Linear &a, hipStream_t st) { return a.pair ? stream<true>(a, st) : stream<false>(a, st); }

}  // namespace lbq
