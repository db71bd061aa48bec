// lbq_kv.hip -- block tables and slot maps from request lengths, and appends to the 8-bit
// paged key/value cache.
#include "lbq_kv.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

namespace lbq {
namespace {

constexpr int STEP_THREADS = 256, STEP_PER = 4, STEP_CHUNK = STEP_THREADS * STEP_PER;

// inclusive sums over the workgroup's threads of two values each
__device__ __forceinline__ void block_scan2(int64_t &a, int64_t &b, int64_t (*sums)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t ua = __shfl_up(a, d), ub = __shfl_up(b, d);
        if (lane >= d) a += ua, b += ub;
    }
    if (lane == 63) sums[wave][0] = a, sums[wave][1] = b;
    __syncthreads();
    for (int w = 0; w < wave; w++) a += sums[w][0], b += sums[w][1];
}

// the last i in [0, n) with v[i] <= x; v never falls and v[0] <= x
__device__ __forceinline__ int last_at_most(const int32_t *v, int n, int32_t x) {
    int lo = 0;
    while (n > 1) {
        const int h = n / 2;
        if (v[lo + h] <= x) lo += h, n -= h;
        else n = h;
    }
    return lo;
}

// Tables, slots and positions of one step.  With n = new_lens, c = ctx_lens, P = page size:
//   cu[b] = n[0] + .. + n[b - 1]          need[b] = ceil((c + n) / P) - ceil(c / P)
//   granted[b]: lengths that fit (table, rows), and need[b] = 0 or need[0] + .. + need[b] <= free
// and the i-th page taken is free_pages[free - 1 - i].  Every workgroup forms the sums over
// all sequences by itself (1024 at a time; the lengths are a few KB and come out of L2), then
// writes its share of the tokens and of the tables: no workgroup reads what another writes,
// so one launch does.  A free count updated in place is written by the last workgroup to
// take a ticket, after all have read it.  The bytes are nothing; bound by latency: lengths, sums, a
// search in LDS, then the old table's entry or the free page.  One token per thread, up to 256
// workgroups: 4.8 us for 16 sequences' tokens, 5.6 for four chunks of up to 512, 8.2 for 22516 tokens of 600 sequences
// (four tokens per thread in turn: 4.8, 6.8, 11.2).
__global__ __launch_bounds__(STEP_THREADS) void k_kv_step(KvStepBuild a) {
    __shared__ int64_t sums[STEP_THREADS / 64][2];
    __shared__ int32_t s_cu[STEP_CHUNK + 1], s_off[STEP_CHUNK + 1], s_ctx[STEP_CHUNK];
    __shared__ uint8_t s_granted[STEP_CHUNK];
    __shared__ int64_t carry[2];
    __shared__ int s_taken;
    const int tid = threadIdx.x, P = 1 << a.log2_page;
    const int64_t stride = (int64_t)gridDim.x * STEP_THREADS, first = (int64_t)blockIdx.x * STEP_THREADS + tid;
    const int32_t count = (int32_t)max((int64_t)0, min((int64_t)*a.free_count, a.num_pages));
    int64_t before_n = 0, before_need = 0;  // sums over the earlier chunks
    int taken = 0;
    if (tid == 0) s_taken = 0;
    for (int base = 0; base < a.batch; base += STEP_CHUNK) {
        const int m = min(STEP_CHUNK, a.batch - base);
        int64_t n[STEP_PER], need[STEP_PER], tn = 0, tneed = 0;
        int32_t ctx[STEP_PER];
        bool fits[STEP_PER];
#pragma unroll
        for (int j = 0; j < STEP_PER; j++) {
            const int i = tid * STEP_PER + j;
            const int32_t c = i < m ? a.ctx_lens[base + i] : 0, w = i < m ? a.new_lens[base + i] : 0;
            const bool ok = c >= 0 && w >= 0;
            const int64_t have = ((int64_t)c + P - 1) >> a.log2_page, want = ((int64_t)c + w + P - 1) >> a.log2_page;
            ctx[j] = c;
            n[j] = ok ? w : 0;
            fits[j] = ok && want <= a.max_blocks && (int64_t)c + w <= INT32_MAX;
            need[j] = fits[j] ? want - have : 0;
            tn += n[j], tneed += need[j];
        }
        // a sequence whose rows do not fit takes no pages: its rows' end is known only
        // after this sum, so the pages are summed again where that happens
        int64_t en = tn, eneed = tneed;
        block_scan2(en, eneed, sums);
        int64_t run = before_n + en - tn;
        tneed = 0;
#pragma unroll
        for (int j = 0; j < STEP_PER; j++) {
            run += n[j];
            if (run > a.num_tokens) fits[j] = false, need[j] = 0;
            tneed += need[j];
        }
        __syncthreads();
        int64_t again = tn;
        eneed = tneed;
        block_scan2(again, eneed, sums);
        int64_t cn = before_n + en - tn, cneed = before_need + eneed - tneed;
#pragma unroll
        for (int j = 0; j < STEP_PER; j++) {
            const int i = tid * STEP_PER + j;
            s_cu[i] = (int32_t)min(cn, a.num_tokens);
            s_off[i] = (int32_t)min(cneed, (int64_t)INT32_MAX);
            cn += n[j], cneed += need[j];
            const bool granted = fits[j] && (need[j] == 0 || cneed <= count);
            s_ctx[i] = ctx[j];
            s_granted[i] = granted;
            if (i < m) {
                if (granted) taken += (int)need[j];
                if (blockIdx.x == 0) {
                    a.seq_lens[base + i] = granted ? ctx[j] + (int32_t)n[j] : 0;
                    a.granted[base + i] = granted;
                    a.cu[base + i] = s_cu[i];
                }
            }
        }
        if (tid == STEP_THREADS - 1) {
            s_cu[STEP_CHUNK] = (int32_t)min(cn, a.num_tokens);
            s_off[STEP_CHUNK] = (int32_t)min(cneed, (int64_t)INT32_MAX);
            carry[0] = cn, carry[1] = cneed;
        }
        __syncthreads();
        // (entries from m on are empty: the searches below pass over them)
        auto page_at = [&](int i, int j) {  // block j of sequence base + i
            const int have = (int)(((int64_t)s_ctx[i] + P - 1) >> a.log2_page);
            return j >= have ? a.free_pages[count - 1 - (s_off[i] + j - have)] : a.tables[(base + i) * a.table_stride + j];
        };
        const int32_t t_end = s_cu[STEP_CHUNK];
        // the first of this thread's tokens in the chunk's range
        const int64_t skip = s_cu[0] > first ? (s_cu[0] - first + stride - 1) / stride : 0;
        for (int64_t t = first + skip * stride; t < t_end; t += stride) {
            const int i = last_at_most(s_cu, m, (int32_t)t);
            int64_t slot = -1;
            int32_t at = -1;
            if (s_granted[i]) {
                at = s_ctx[i] + ((int32_t)t - s_cu[i]);
                const int32_t page = page_at(i, at >> a.log2_page);
                if (page >= 0 && page < a.num_pages) slot = ((int64_t)page << a.log2_page) + (at & (P - 1));
                else at = -1;
            }
            a.slots[t] = slot;
            a.positions[t] = at;
        }
        const int32_t p_end = min(s_off[STEP_CHUNK], count);
        const int64_t skip_p = s_off[0] > first ? (s_off[0] - first + stride - 1) / stride : 0;
        for (int64_t p = first + skip_p * stride; p < p_end; p += stride) {
            const int i = last_at_most(s_off, m, (int32_t)p);
            if (!s_granted[i]) continue;
            const int have = (int)(((int64_t)s_ctx[i] + P - 1) >> a.log2_page);
            a.tables[(base + i) * a.table_stride + have + ((int32_t)p - s_off[i])] = a.free_pages[count - 1 - p];
        }
        before_n = carry[0], before_need = carry[1];
        __syncthreads();
    }
    // rows behind the last sequence
    const int64_t total = min(before_n, a.num_tokens), skip = total > first ? (total - first + stride - 1) / stride : 0;
    for (int64_t t = first + skip * stride; t < a.num_tokens; t += stride) a.slots[t] = -1, a.positions[t] = -1;
    if (taken) atomicAdd(&s_taken, taken);  // whole numbers: any order
    __syncthreads();
    if (tid == 0) {
        if (blockIdx.x == 0) a.cu[a.batch] = (int32_t)total;
        if (a.free_count_out != a.free_count) {
            if (blockIdx.x == 0) *a.free_count_out = count - s_taken;
        } else {
            __threadfence();
            if (gridDim.x == 1 || atomicAdd(a.ticket, 1u) == gridDim.x - 1) {
                *a.free_count_out = count - s_taken;
                if (gridDim.x > 1) *a.ticket = 0;
            }
        }
    }
}

// The pages of the sequences with which[b] != 0 go back on top of the free pages, in the order of
// the sequences and of their blocks; their table entries become -1.  One workgroup: few sequences
// end in a step, and the order is then the same every time.  The entries of 1024 sequences form one list,
// of which each thread takes every 1024th: a list position's sequence is found in the running sums
// of their blocks.  Bound by latency, a table entry and two barriers for each 1024 entries: 4.3 us for 16
// sequences of 64 pages, 60 us for 600 (sequence by sequence: 14 and 524; one sequence 2.7 instead of 4.1).
__global__ __launch_bounds__(1024) void k_kv_release(KvRelease a) {
    __shared__ int64_t starts[1024];
    __shared__ int64_t s_sums[16];
    __shared__ int s_waves[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = 1 << a.log2_page;
    int64_t count = max((int64_t)0, min((int64_t)*a.free_count, a.num_pages));
    for (int base = 0; base < a.batch; base += 1024) {
        const int b = base + tid;
        int64_t blocks = 0;
        if (b < a.batch && a.which[b] != 0 && a.lens[b] > 0) blocks = min((int64_t)a.max_blocks, ((int64_t)a.lens[b] + P - 1) >> a.log2_page);
        int64_t sum = blocks;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int64_t up = __shfl_up(sum, d);
            if (lane >= d) sum += up;
        }
        if (lane == 63) s_sums[wave] = sum;
        __syncthreads();
        int64_t total = 0;
        for (int w = 0; w < 16; w++) {
            if (w < wave) sum += s_sums[w];
            total += s_sums[w];
        }
        starts[tid] = sum - blocks;
        __syncthreads();
        for (int64_t e0 = 0; e0 < total; e0 += 1024) {
            const int64_t e = e0 + tid;
            int32_t *entry = nullptr;
            int32_t page = -1;
            if (e < total) {
                int row = 0;  // the last that starts at or before e (those without blocks are passed over)
#pragma unroll
                for (int h = 512; h; h /= 2)
                    if (starts[row + h] <= e) row += h;
                entry = a.tables + (base + row) * a.table_stride + (e - starts[row]);
                page = *entry;
            }
            const bool keep = page >= 0 && page < a.num_pages;
            const uint64_t kept = __ballot(keep);
            if (lane == 0) s_waves[wave] = __popcll(kept);
            __syncthreads();
            int64_t to = count + __popcll(kept & ((1ull << lane) - 1)), all = 0;
            for (int w = 0; w < 16; w++) {
                if (w < wave) to += s_waves[w];
                all += s_waves[w];
            }
            if (keep && to < a.num_pages) a.free_pages[to] = page;
            if (entry) *entry = -1;
            count = min(count + all, a.num_pages);
            __syncthreads();
        }
        __syncthreads();
    }
    if (tid == 0) *a.free_count = (int32_t)count;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ float load_value(const void *p, int64_t i) {
    if constexpr (DT == DT_F32) return static_cast<const float *>(p)[i];
    else if constexpr (DT == DT_F16) return __half2float(static_cast<const __half *>(p)[i]);
    else return __uint_as_float((uint32_t) static_cast<const uint16_t *>(p)[i] << 16);
}
template <int DT>
__device__ __forceinline__ void store_value(void *p, int64_t i, float v) {
    if constexpr (DT == DT_F32) static_cast<float *>(p)[i] = v;
    else if constexpr (DT == DT_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__hip_bfloat16 *>(p)[i] = __float2bfloat16(v);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// four neighbouring values, at an address that is a multiple of their size
template <int DT>
__device__ __forceinline__ f32x4 load4(const void *p, int64_t i) {
    if constexpr (DT == DT_F32) {
        return *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i);
    } else {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + i);
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint16_t h = (uint16_t)(w[j / 2] >> (16 * (j % 2)));
            v[j] = load_value<DT>(&h, 0);
        }
        return v;
    }
}
template <int DT>
__device__ __forceinline__ void store4(void *p, int64_t i, f32x4 v) {
    if constexpr (DT == DT_F32) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(p) + i) = v;
    } else {
        uint16_t h[4];
#pragma unroll
        for (int j = 0; j < 4; j++) store_value<DT>(h, j, v[j]);
        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p) + i) = u32x2{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
    }
}

// The pair (x, y) rotated: (x c - y s, y c + x s).  Both products are exact in 64 bits and their sum
// is rounded once there and once to 32: one value whatever the order, which the codes need (a
// last bit moves a code that lies at a tie).
__device__ __forceinline__ void rotate_pair(float x, float y, float c, float s, float &u, float &w) {
    u = (float)((double)x * c - (double)y * s);
    w = (float)((double)y * c + (double)x * s);
    // (the compiler would round a 16-bit result from 64 bits at once: another value at some ties)
    asm("" : "+v"(u), "+v"(w));
}

// Eight channels of a row, rotated where they are among the first rot_dim: `at` gets the first channel
// of each four of them.  Unit u of a row is channels 8 u and on; where pairs lie half a row apart, the
// rotated ones' units are four channels of either half.  A position outside the table gives NaN.
template <int DT, bool VEC>
__device__ __forceinline__ void load_unit(const KvAppend &a, const void *row, int u, int64_t pos, bool turn, f32x4 v[2], int at[2]) {
    const int half = a.rot_dim / 2;
    at[0] = 8 * u, at[1] = 8 * u + 4;
    if constexpr (VEC) {
        const bool mine = turn && u < a.rot_dim / 8;
        if (mine && !a.interleaved) at[0] = 4 * u, at[1] = 4 * u + half;
        const f32x4 x = load4<DT>(row, at[0]), y = load4<DT>(row, at[1]);
        v[0] = x, v[1] = y;
        if (!mine) return;
        if (pos < 0 || pos >= a.max_pos) {
            v[0] = v[1] = f32x4{1.f, 1.f, 1.f, 1.f} * __uint_as_float(0x7fc00000u);
            return;
        }
        const f32x4 c = *reinterpret_cast<const f32x4 *>(a.cos + pos * half + 4 * u), s = *reinterpret_cast<const f32x4 *>(a.sin + pos * half + 4 * u);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float p, q;
            if (a.interleaved) {
                const f32x4 &z = j < 2 ? x : y;
                rotate_pair(z[2 * (j % 2)], z[2 * (j % 2) + 1], c[j], s[j], p, q);
                v[j / 2][2 * (j % 2)] = p, v[j / 2][2 * (j % 2) + 1] = q;
            } else {
                rotate_pair(x[j], y[j], c[j], s[j], p, q);
                v[0][j] = p, v[1][j] = q;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int d = 8 * u + j;
            float x = load_value<DT>(row, d);
            if (turn && d < a.rot_dim) {
                if (pos < 0 || pos >= a.max_pos) {
                    x = __uint_as_float(0x7fc00000u);
                } else {
                    const int i = a.interleaved ? d / 2 : d < half ? d : d - half;
                    const bool second = a.interleaved ? d & 1 : d >= half;
                    const float y = load_value<DT>(row, a.interleaved ? d ^ 1 : second ? d - half : d + half);
                    float p, q;
                    rotate_pair(second ? y : x, second ? x : y, a.cos[pos * half + i], a.sin[pos * half + i], p, q);
                    x = second ? q : p;
                }
            }
            v[j / 4][j % 4] = x;
        }
    }
}

// The scale of a block whose largest magnitude is amax: int8 amax / 127; e4m3 the power of
// two that brings amax to at most 448 (a floating code loses nothing by it, and x / scale is
// exact).  Never below the smallest normal number; NaN where a value is not finite.
__device__ __forceinline__ float block_scale(float amax, int kind) {
    if (!(amax < INFINITY)) return __uint_as_float(0x7fc00000u);
    if (amax == 0.f) return 0.f;
    if (kind == KV_INT8) return fmaxf(amax / 127.f, 0x1p-126f);
    int e;
    const float m = frexpf(amax, &e);
    return ldexpf(1.f, max(m > 0.875f ? e - 8 : e - 9, -126));
}

// x / s to the nearest code, ties to even, decided as if the quotient were exact; 0 where s is 0
// or NaN.  inv: 1 / s.
__device__ __forceinline__ uint32_t code_of(float x, float s, float inv, int kind) {
    if (kind == KV_E4M3) return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x * inv, 0.f, 0, false) & 0xffu;  // (a power of two: exact)
    // rint of the product is the answer or, next to a tie, one beside it; what is left, x - q s, is
    // exact in f32 (a multiple of the operands' last place no larger than about s), so its
    // comparison with s / 2 decides
    const float q = rintf(x * inv), left = fmaf(-q, s, x), most = 0.5f * s;
    const int i = (int)q;
    const bool move = fabsf(left) > most || (fabsf(left) == most && (i & 1));
    return (uint32_t)(move ? left > 0.f ? i + 1 : i - 1 : i) & 0xffu;
}

// a code under scale `was`, under the larger scale `now`
__device__ __forceinline__ uint8_t recode(uint8_t c, float was, float now, int kind) {
    if (kind == KV_E4M3)  // a power of two: exact up to the one rounding
        return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8((int)c, 0) * (was / now), 0.f, 0, false);
    return (uint8_t)(int8_t)(int)rint((double)(int8_t)c * (double)was / (double)now);
}

constexpr int APPEND_THREADS = 256;

// One workgroup per (run of new tokens in one page, kv head, keys or values); the workgroups
// behind those rotate queries.  Bound by reading q, k and v and writing q: eight channels of a
// row per thread at a time, in 16-byte accesses where the tensors allow (VEC).
//
// Sequence b has at most cu[b + 1] / P - cu[b] / P + 2 runs, so run r belongs to the sequence with
// cu[b] / P + 2 b <= r, without a list.  The new values are rotated into LDS while their largest
// magnitude is found, then coded from there, 16 codes per store: keys along the channels, values
// along the tokens.  A scale never falls while a page fills; where it grows, the codes that are
// there are coded again, through a table of all 256.  One workgroup owns a (page, head)'s
// codes and scale: no atomics.  5.9 us for one token or 64 (latency: rows' bounds, slot, values, code),
// 15 us for four chunks of 512 tokens of 32 + 8 + 8 heads in f32, 67.9 MB at 4.5 TB/s, where a large copy runs at 5.0
// (one channel per thread and single-byte stores of codes: 46).
template <int DT, bool VEC>
__global__ __launch_bounds__(APPEND_THREADS) void k_kv_append(KvAppend a, int runs) {
    extern __shared__ __align__(16) float vals[];
    __shared__ float s_max[APPEND_THREADS / 64];
    __shared__ uint8_t s_again[256];
    const int tid = threadIdx.x, threads = blockDim.x, D = a.c.head_dim, P = a.c.page_size, H = a.c.kv_heads;
    constexpr int size = DT == DT_F32 ? 4 : 2;
    const int units = D / 8, u = tid % units, step = threads / units, first = tid / units;  // (threads from step * units on: idle)
    const int64_t id = blockIdx.x, kv_groups = (int64_t)runs * H * 2;
    if (id >= kv_groups) {
        const int64_t n = a.s.num_tokens * a.q_heads, stride = (gridDim.x - kv_groups) * step;
        if (first >= step) return;
        for (int64_t row = (id - kv_groups) * step + first; row < n; row += stride) {
            const uint32_t t = (uint32_t)row / (uint32_t)a.q_heads, h = (uint32_t)row % (uint32_t)a.q_heads;
            const int32_t pos = a.s.positions[t];
            if (pos < 0) continue;
            f32x4 v[2];
            int at[2];
            load_unit<DT, VEC>(a, static_cast<const char *>(a.q.p) + (t * a.q.token_stride + h * a.q.head_stride) * size, u, pos, a.rot_dim > 0, v, at);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if constexpr (VEC) {
                    store4<DT>(a.q_out, row * D + at[j], v[j]);
                } else {
#pragma unroll
                    for (int z = 0; z < 4; z++) store_value<DT>(a.q_out, row * D + at[j] + z, v[j][z]);
                }
            }
        }
        return;
    }
    const bool is_v = id & 1;
    const int h = (int)((id >> 1) % H);
    const int64_t run = (id >> 1) / H;
    const int b = find_sequence(a.s.batch, run, [&](int i) { return (int64_t)(a.s.cu[i] >> a.c.log2_page) + 2 * (int64_t)i; });
    const int64_t t0 = a.s.cu[b], t1 = a.s.cu[b + 1], len = a.s.seq_lens[b], ctx = len - (t1 - t0);
    if (t0 < 0 || t1 > a.s.num_tokens || t1 <= t0 || ctx < 0) return;
    if (a.max_new > 0 && t1 - t0 > a.max_new) return;  // (LDS is for no more)
    const int64_t block = (ctx >> a.c.log2_page) + run - ((t0 >> a.c.log2_page) + 2 * (int64_t)b);
    const int64_t lo = max(block << a.c.log2_page, ctx), hi = min((block + 1) << a.c.log2_page, len);
    if (lo >= hi) return;
    const int64_t tok = t0 + (lo - ctx), slot = a.s.slots[tok], page = slot >> a.c.log2_page;
    const int o = (int)(lo & (P - 1)), count = (int)(hi - lo);
    if (slot < 0 || page >= a.c.num_pages || (int)(slot & (P - 1)) != o) return;

    const KvRows &rows = is_v ? a.v : a.k;
    float *const sp = (is_v ? a.c.vs : a.c.ks) + page * H + h;
    const float was = o ? *sp : 0.f;
    float amax = 0.f;
    bool bad = false;
    if (first < step)
        for (int j = first; j < count; j += step) {
            const void *row = static_cast<const char *>(rows.p) + ((tok + j) * rows.token_stride + h * rows.head_stride) * size;
            const bool turn = !is_v && a.rot_dim > 0;
            f32x4 v[2];
            int at[2];
            load_unit<DT, VEC>(a, row, u, turn ? a.s.positions[tok + j] : 0, turn, v, at);
#pragma unroll
            for (int z = 0; z < 2; z++) {
                *reinterpret_cast<f32x4 *>(vals + j * D + at[z]) = v[z];
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    bad |= !(fabsf(v[z][y]) < INFINITY);
                    amax = fmaxf(amax, fabsf(v[z][y]));
                }
            }
        }
    if (bad) amax = INFINITY;
#pragma unroll
    for (int d = 32; d; d /= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
    if ((tid & 63) == 0) s_max[tid >> 6] = amax;
    __syncthreads();
    for (int w = 0; w < threads / 64; w++) amax = fmaxf(amax, s_max[w]);
    const float fresh = block_scale(amax, a.c.kind);
    const float now = was != was || fresh != fresh ? __uint_as_float(0x7fc00000u) : fmaxf(was, fresh);
    uint8_t *const codes = (is_v ? a.c.v : a.c.k) + (page * H + h) * (int64_t)P * D;
    if (now > was && was > 0.f) {  // (the same in every thread)
        for (int i = tid; i < 256; i += threads) s_again[i] = recode((uint8_t)i, was, now, a.c.kind);
        __syncthreads();
        // whole 16-byte pieces that hold a code from before; what else is in one stays, or is
        // written below
        const int pieces = is_v ? D * ((o + 15) / 16) : o * D / 16, per_row = (o + 15) / 16;
        for (int i = tid; i < pieces; i += threads) {
            u32x4 *const to = reinterpret_cast<u32x4 *>(codes + (is_v ? i / per_row * P + i % per_row * 16 : i * 16));
            const int keep = is_v ? o - i % per_row * 16 : 16;
            u32x4 w = *to;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const uint32_t c = w[j / 4] >> (8 * (j % 4)) & 0xffu;
                if (j < keep) w[j / 4] = (w[j / 4] & ~(0xffu << (8 * (j % 4)))) | (uint32_t)s_again[c] << (8 * (j % 4));
            }
            *to = w;
        }
        __syncthreads();
    }
    const bool none = !(now > 0.f);  // a scale of 0 or NaN: all codes are 0
    const float inv = none ? 0.f : 1.f / now, s = none ? 0.f : now;
    if (!is_v) {
        for (int i = tid; i < count * D / 16; i += threads) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(vals + 16 * i + 4 * j);
                w[j] = none ? 0u
                            : code_of(x[0], s, inv, a.c.kind) | code_of(x[1], s, inv, a.c.kind) << 8 | code_of(x[2], s, inv, a.c.kind) << 16 |
                                  code_of(x[3], s, inv, a.c.kind) << 24;
            }
            *reinterpret_cast<u32x4 *>(codes + o * D + 16 * i) = w;
        }
    } else {
        // channel i mod D, places 16 (o / 16 + i / D) and on: a lane's neighbours read neighbours of one token
        const int g0 = o / 16, groups = (o + count + 15) / 16 - g0;
        for (int i = tid; i < groups * D; i += threads) {
            const int d = i % D, at = 16 * (g0 + i / D);
            const int from = max(o - at, 0), to = min(o + count - at, 16);
            uint8_t *const out = codes + d * P + at;
            if (from == 0 && to == 16) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t c = 0;
#pragma unroll
                    for (int z = 0; z < 4; z++) c |= code_of(vals[(at - o + 4 * j + z) * D + d], s, inv, a.c.kind) << (8 * z);
                    w[j] = none ? 0u : c;
                }
                *reinterpret_cast<u32x4 *>(out) = w;
            } else {
                for (int j = from; j < to; j++) out[j] = none ? 0 : (uint8_t)code_of(vals[(at - o + j) * D + d], s, inv, a.c.kind);
            }
        }
    }
    if (tid == 0) *sp = now;
}

}  // namespace

hipError_t launch_kv_step(const KvStepBuild &a, hipStream_t st) {
    const int64_t groups = std::max<int64_t>(1, std::min<int64_t>((a.num_tokens + STEP_THREADS - 1) / STEP_THREADS, 256));
    k_kv_step<<<dim3((unsigned)groups), STEP_THREADS, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_release(const KvRelease &a, hipStream_t st) {
    k_kv_release<<<1, 1024, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppend &a, hipStream_t st) {
    const int D = a.c.head_dim;
    const int64_t runs = std::min<int64_t>((a.s.num_tokens >> a.c.log2_page) + 2 * (int64_t)a.s.batch, INT32_MAX);
    const int rows = a.max_new > 0 ? std::min(a.max_new, a.c.page_size) : a.c.page_size;
    // one wave where the largest run has no work for more
    const int threads = rows * (D / 8) <= 64 ? 64 : APPEND_THREADS, step = threads / (D / 8);
    const int64_t q = a.q.p ? std::min<int64_t>((a.s.num_tokens * a.q_heads + 2 * step - 1) / (2 * step), 65536) : 0;  // two rows a thread
    const size_t lds = (size_t)rows * D * sizeof(float);
    const unsigned align = a.dtype == DT_F32 ? 16 : 8;
    auto whole = [&](const KvRows &r) { return !r.p || (reinterpret_cast<uintptr_t>(r.p) % align == 0 && r.token_stride % 4 == 0 && r.head_stride % 4 == 0); };
    const bool vec = whole(a.q) && whole(a.k) && whole(a.v) && reinterpret_cast<uintptr_t>(a.q_out) % align == 0 && a.rot_dim % 8 == 0 &&
                     reinterpret_cast<uintptr_t>(a.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(a.sin) % 16 == 0;
    auto pick = [&](auto with, auto without) { return vec ? with : without; };
    auto k = a.dtype == DT_F32   ? pick(k_kv_append<DT_F32, true>, k_kv_append<DT_F32, false>)
             : a.dtype == DT_F16 ? pick(k_kv_append<DT_F16, true>, k_kv_append<DT_F16, false>)
                                 : pick(k_kv_append<DT_BF16, true>, k_kv_append<DT_BF16, false>);
    if (lds > 65536 - 1024) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    k<<<dim3((unsigned)(runs * a.c.kv_heads * 2 + q)), threads, lds, st>>>(a, (int)runs);
    return hipGetLastError();
}

}  // namespace lbq
