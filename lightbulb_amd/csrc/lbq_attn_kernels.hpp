// lbq_attn_kernels.hpp -- attention over the 8-bit paged key/value cache on the f16 matrix cores.
//
// The codes of both kinds are f16 numbers, so a code goes into a matrix instruction exactly and
// its scale, one per 16 or more keys, into the f32 logit or weight.  f32 queries go in as two f16
// parts of a power-of-two multiple of their row (22 bits, and no less than 2^-40 of the row's largest); f16 and bf16
// queries are one part, exactly down to 2^-28 of it.  (int8 keys of the short form: attn_short.)
// Weights go in as two f16 parts, for bf16 as one.  The products of both parts go into one f32 sum:
// results of f32's accuracy at twice the matrix work.
//
// Products are formed transposed: S^T = K Q^T, then O^T = V^T P^T.  Column n of every tile is
// query row n, so a row's softmax stays inside a lane and the lanes that share its column, and the
// accumulator layout of S^T (column = lane mod 16 or 32, rows in registers) is already the operand
// layout of P^T once the rows of K are taken in the right order.  Weights never leave registers.
//
// Value scales are applied to the weights, inside the exponential: a weight is 2^(x + s - b), x the logit
// and 2^s the key's value scale relative to a power of two r that no scale seen so far exceeds.  Its base b
// follows the row's largest x + s, not its largest x, so that what decides the row's result is held to the
// same bits whatever other pages' scales are: seen with no weight, or by other rows only.  b is moved only when
// the maximum is 2^6 above it (moving it multiplies all accumulators).  Weights carry a factor 2^9, so
// that they stay below 2^15 and both f16 parts of those that matter clear of the subnormals.  The row's sum
// is that of 2^(x - b) with the same factor.
#pragma once
#include "lbq_kv.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

namespace lbq {

// the launch's plan, the same in the kernels and in the join
struct AttnPlan {
    int splits_short, splits_long;  // parts that a sequence's keys are cut into
    // Rows of parts: [splits_short][short_tokens][q_heads] of the short form from row 0, then
    // [splits_long][num_q][q_heads] of the long form from row long_row on.  A short sequence's tokens
    // are those of the batch, or short_per for each sequence where that is fewer (a prompt's rows have
    // no place among the parts of a single token's long context).
    float *part;                    // [rows][head_dim]: outputs of parts
    float *stat;                    // [rows][2]: running maximum (log2), sum
    int64_t short_tokens, long_row;
    int short_per;                  // 0: the batch's tokens
    int tiles;                      // tiles of the long form, an upper bound
    int tiles_per;                  // no sequence has more tiles than these; 0: not known
    int short_groups;               // tiles of the short form (16 rows), an upper bound
    int short_tiles;                // of each sequence, likewise
    int listed;                     // whether sequences and tiles are counted on the device, without those of another form
    int group;                      // query heads per kv head
    int short_rows;                 // rows (queries * group) up to which a sequence takes the short form; 0: none does
};

namespace attn {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int SHORT_ROWS = 16;  // rows of one kv head's queries in a tile of the short form
constexpr int TILE = 64;  // keys per step of either form

// f16 parts of a query value and of a weight.  f16 outputs take weights of two parts too: one
// part's rounding is as large as the output's own, and would leave it 1.4 times as far off.  bf16 outputs
// take one: their own rounding is 16 times as large (the 8000-token prompt: 471 us and 0.00166 off the definition in 64
// bits; with two parts 604 us and 0.00165, as 32-bit arithmetic has it; one value in ten is rounded to the neighbour instead).
template <int DT>
constexpr int QUERY_PARTS = DT == DT_F32 ? 2 : 1;
template <int DT>
constexpr int WEIGHT_PARTS = DT == DT_BF16 ? 1 : 2;

template <int DT>
__device__ __forceinline__ float load_value(const void *p, int64_t i) {
    if constexpr (DT == DT_F32) return static_cast<const float *>(p)[i];
    else if constexpr (DT == DT_F16) return __half2float(static_cast<const __half *>(p)[i]);
    else return __uint_as_float((uint32_t) static_cast<const uint16_t *>(p)[i] << 16);
}
template <int DT>
__device__ __forceinline__ void store_values4(void *p, int64_t i, const float *v) {
    if constexpr (DT == DT_F32) {
        // (a contiguous output's rows of 64 or more values need no more than their own 4-byte alignment)
        float *o = static_cast<float *>(p) + i;
        o[0] = v[0], o[1] = v[1], o[2] = v[2], o[3] = v[3];
    } else if constexpr (DT == DT_F16) {
        _Float16 *o = static_cast<_Float16 *>(p) + i;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = (_Float16)v[j];
    } else {
        __hip_bfloat16 *o = static_cast<__hip_bfloat16 *>(p) + i;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = __float2bfloat16(v[j]);
    }
}

// weights carry 2^WEIGHT_LOG2, and their base is moved when the maximum is LAZY_LOG2 above it
constexpr float WEIGHT_LOG2 = 9.f, LAZY_LOG2 = 6.f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// the larger of two, one instruction (fmaxf of values whose origin the compiler does not know takes three)
__device__ __forceinline__ float larger(float x, float y) { return __builtin_amdgcn_fmed3f(x, y, INFINITY); }
// a maximum as the base of exponents: 0 where nothing was seen, so that no inf - inf is formed
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// four codes of a word as f16, exactly.  int8: the byte + 128 under the exponent of 1024, less 1152.
template <int KIND>
__device__ __forceinline__ half4 codes4(uint32_t w) {
    if constexpr (KIND == KV_INT8) {
        const uint32_t x = w ^ 0x80808080u;
        const half2v off = {(_Float16)-1152.f, (_Float16)-1152.f};
        const half2v a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + off;
        const half2v b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + off;
        return half4{a[0], a[1], b[0], b[1]};
    } else {
        const half2v a = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, false));
        const half2v b = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, true));
        return half4{a[0], a[1], b[0], b[1]};
    }
}
template <int KIND>
__device__ __forceinline__ half8 codes8(uint32_t lo, uint32_t hi) {
    return __builtin_shufflevector(codes4<KIND>(lo), codes4<KIND>(hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// the first `keep` (0 .. 16) of 16 code bytes, zeros behind them
__device__ __forceinline__ u32x4 keep_bytes(u32x4 v, int keep) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int n = min(max(keep - 4 * i, 0), 4);
        v[i] &= n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
    }
    return v;
}

// eight f32 values as one f16 operand, or two that add up to them
template <int NS>
__device__ __forceinline__ void parts8(const float *v, half8 *o) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const half2v hi = __builtin_convertvector((f32x2){v[j], v[j + 1]}, half2v);
        o[0][j] = hi[0], o[0][j + 1] = hi[1];
        if constexpr (NS == 2) {
            // v - hi, exactly, taking the f16 as it is (the compiler widens it first)
            float d0, d1;
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d0) : "v"(hi), "v"(v[j]));
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d1) : "v"(hi), "v"(v[j + 1]));
            const half2v lo = __builtin_convertvector((f32x2){d0, d1}, half2v);
            o[NS - 1][j] = lo[0], o[NS - 1][j + 1] = lo[1];
        }
    }
}

// Four values as whole numbers of four signed digits to the base of 256: o[i] has digit i of each
// (256^3 o[3] + 256^2 o[2] + 256 o[1] + o[0]).  With the row's largest in 31 bits what is 2^-8 of it still has all
// the bits of an f32, and nothing is off by more than 2^-31 of it (three digits, 2^-24: a channel a thousand times
// the others left them 14 bits).
constexpr float MOST_DIGITS = 0x7f7f7f00;  // the largest f32 up to 127 in each digit
__device__ __forceinline__ void digits4(const float *v, uint32_t *o) {
    uint32_t w[4];  // the number + 128 in each digit
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = (uint32_t)(int)rintf(v[j]) + 0x80808080u;
#pragma unroll
    for (int i = 0; i < 2; i++) {  // digits 2 i and 2 i + 1
        const uint32_t pick = i ? 0x07030602u : 0x05010400u;
        const uint32_t ab = __builtin_amdgcn_perm(w[1], w[0], pick), cd = __builtin_amdgcn_perm(w[3], w[2], pick);
        o[2 * i] = __builtin_amdgcn_perm(cd, ab, 0x05040100u) ^ 0x80808080u;
        o[2 * i + 1] = __builtin_amdgcn_perm(cd, ab, 0x07060302u) ^ 0x80808080u;
    }
}

// the exponent e with |max| < 2^e for the parts of a query row: values times 2^(15 - e) fit f16
__device__ __forceinline__ int row_exponent(float amax) {
    int e = 0;
    if (amax > 0.f && amax < INFINITY) (void)frexpf(amax, &e);
    return e;
}

// the exponent of a power of two no smaller than a value scale (and normal, as is its inverse)
__device__ __forceinline__ int scale_ceiling(float s) { return min(max(__builtin_amdgcn_frexp_expf(s), -126), 126); }

// what a sequence's rows see, and where its queries lie
struct Sequence {
    int t0;     // first query row
    int n;      // its queries
    int len;    // keys that can be seen at all
    int first;  // position of the first query
};
__device__ __forceinline__ bool sequence_of(const KvAttention &a, int b, Sequence &s) {
    const int t0 = a.cu_q[b], t1 = a.cu_q[b + 1];
    if (t0 < 0 || t1 > a.num_q || t1 <= t0) return false;
    s.t0 = t0;
    s.n = t1 - t0;
    const int len = max(a.s.seq_lens[b], 0);
    s.len = min(len, a.max_len);
    s.first = len - s.n;
    return true;
}

// Item x of a list that holds count(i) items of each sequence i in order, for up to LISTED sequences:
// its sequence and its place among that one's; or, where `last` is set, the x-th item from the end.  The same
// x in every lane of a wave; all 64 lanes call it.
constexpr int LISTED = 256;
template <class Count>
__device__ __forceinline__ bool find_item(int batch, int x, bool last, Count count, int &b, int &index) {
    constexpr int PER = LISTED / 64;
    const int lane = threadIdx.x & 63;
    int c[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        c[j] = lane * PER + j < batch ? count(lane * PER + j) : 0;
        sum += c[j];
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int before = __shfl_up(upto, d);
        if (lane >= d) upto += before;
    }
    const int total = __builtin_amdgcn_readlane(upto, 63);
    if (x >= total) return false;
    if (last) x = total - 1 - x;
    const int at = __popcll(__ballot(upto <= x));  // (sums never fall: the lanes before the item's)
    index = x - __builtin_amdgcn_readlane(upto - sum, at);
    b = at * PER;
    bool found = false;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int n = __builtin_amdgcn_readlane(c[j], at);
        found |= index < n;
        if (!found) index -= n, b++;
    }
    return true;
}

// The same where each sequence holds one item or none: by counting bits alone.
template <class Has>
__device__ __forceinline__ bool find_one(int batch, int x, bool last, Has has, int &b) {
    constexpr int PER = LISTED / 64;
    const int lane = threadIdx.x & 63;
    uint64_t mask[PER], in = 0;
    int total = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        mask[j] = __ballot(64 * j + lane < batch && has(64 * j + lane));
        total += __popcll(mask[j]);
    }
    if (x >= total) return false;
    if (last) x = total - 1 - x;
    b = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int n = __popcll(mask[j]);
        if (in) continue;
        if (x < n) in = mask[j], b = 64 * j;
        else x -= n;
    }
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
    b += __ffsll((unsigned long long)__ballot((in >> lane & 1) && before == x)) - 1;
    return true;
}

// keys [lo, hi) that the query at position pos sees
__device__ __forceinline__ void seen_range(const KvAttention &a, const Sequence &s, int pos, int &lo, int &hi) {
    hi = a.causal ? max(min(s.len, pos + 1), 0) : s.len;
    lo = a.causal && a.window > 0 ? max(pos - a.window + 1, 0) : 0;
}

// x, or -infinity where j is outside [from, to).  On the vector unit alone: compares would hold a
// pair of scalar registers for each value, and there are none left.
__device__ __forceinline__ float seen_or_not(float x, int j, int from, int to) {
    const uint32_t out = (uint32_t)(((j - from) | (to - 1 - j)) >> 31);
    return __uint_as_float((out & 0xff800000u) | (~out & __float_as_uint(x)));
}

// The weights' factor for a value scale s, relative to r and in powers of two.  A scale below 2^-80 r, or of 0,
// counts as that.  So no logit of a row is more than 86 above b (which is at most 6 behind the logit less 80):
// a row's sum stays below 2^95 for each key.  And b is no more than the largest logit: a key that matters to
// the sum, 2^-30 of it say, has a weight of at least 2^(9 - 30 - 80), a normal number.
// (The last term is 0, or NaN for a scale that is.)
__device__ __forceinline__ float scale_log(float s, float inv_r) {
    return fmaf(s, 0.f, fmaxf(__builtin_amdgcn_logf(s * inv_r), -80.f));
}

// what a row's weights are relative to, in powers of two
struct Base {
    float b = -INFINITY;
    float r = 0.f, inv_r = 1.f;

    // r grows to 2^e and b falls as much, but no lane's part l of the row's sum (the largest: row_l) passes 2^100 by
    // it: the outputs' factor, 1 (or what the rounding of b leaves) unless the sum keeps b up.  Outputs under
    // scales of 0 stand for nothing.
    __device__ __forceinline__ float grow(int e, float &l, float row_l) {
        const float by = (float)(e + 1 - __builtin_amdgcn_frexp_expf(r)), most = fmaxf((float)(100 - __builtin_amdgcn_frexp_expf(row_l)), 0.f);
        const float to = b - (r == 0.f ? most : fminf(by, most)), fall = b == -INFINITY ? 0.f : b - to;
        const float factor = r == 0.f ? 0.f : exp2_fast(fall - by);
        l *= exp2_fast(fall);
        b = to;
        r = ldexpf(1.f, e), inv_r = ldexpf(1.f, -e);
        return factor;
    }
    // the largest logit with its scale is `top`, or it was: the factor of sum and outputs
    __device__ __forceinline__ float move(float top) {
        const float to = fmaxf(b, top), factor = exp2_fast(b - base_of(to));
        b = to;
        return factor;
    }
};
// a row's sum, whose exponent goes into its base, for joins: at most 1 (m + e is rounded, its difference from m is not)
__device__ __forceinline__ void settle(float &m, float &l) {
    if (!(l > 0.f && l < INFINITY)) return;
    const float to = m + (float)__builtin_amdgcn_frexp_expf(l);
    l *= exp2_fast(m - to);
    m = to;
}

// A logit's factor where products of -infinity stand for keys that are not seen: not 0, which
// would make them NaN.  (What it multiplies besides is below 2^39.)
__device__ __forceinline__ float not_zero(float f) { return f == 0.f ? 0x1p-126f : f; }

// The join of parts' outputs o_i with maxima m_i and sums l_i: weights l_i 2^(m_i - max).
__device__ __forceinline__ float part_weight(float m, float l, float top) { return l * exp2_fast(m - base_of(top)); }

// ---------------------------------------------------------------------------
// Short form: tiles of up to 16 query rows of one kv head (a token step: its group of query heads).
// Bound by reading the cache, 2 head_dim bytes per key: one wave takes 64 keys at a time
// straight from memory into its operands, the next 64 on their way while it works, with no
// barrier until the waves' outputs are joined at the end.  32 tokens of 8 heads with ragged contexts
// of up to 4096 keys of 128 channels, 202.7 MB: 45 us, 4.5 TB/s (a read stream reaches 5.7; here 256
// workgroups of unlike length start and end apart).  131071 keys of one sequence, 268 MB: 51 us, 5.3 TB/s,
// and 4 to join 32 parts.  One workgroup takes 2.5 us for a step of its eight waves, most of it the
// values' way to f16 and the weights, and 7 for launch, bounds, pages and the first codes: a short context's
// time (1000 keys: 12.3 us).  16x16x32 products; in S^T lane
// (c, n) = (lane / 16, lane % 16) holds keys 16 c .. 16 c + 15 of the 64 for row n, which is
// what the products with V take, and all of one page: one scale per lane.
// ---------------------------------------------------------------------------
template <int D, int WAVES>
constexpr size_t short_lds() { return sizeof(float) * WAVES * SHORT_ROWS * (D + 4 + 2); }

// group: its place among the form's workgroups (parts * kv heads * tiles); lds: short_lds bytes
template <int D, int KIND, int DT, int WAVES>
__device__ __forceinline__ void attn_short(const KvAttention &a, const AttnPlan &plan, int group, float *lds) {
    constexpr int NS = QUERY_PARTS<DT>, NW = WEIGHT_PARTS<DT>;
    constexpr int STEPS = D / 32, DB = D / 16;
    // int8 keys need not go to f16: with the row as whole numbers of four digits the products are
    // whole too, and exact (32 tokens: 44.9 us, with f16 keys 46.3; at 500 keys 9.6 and 9.7)
    constexpr bool DIGITS = KIND == KV_INT8;
    float(*const s_o)[SHORT_ROWS][D + 4] = reinterpret_cast<float(*)[SHORT_ROWS][D + 4]>(lds);
    float(*const s_m)[SHORT_ROWS] = reinterpret_cast<float(*)[SHORT_ROWS]>(lds + WAVES * SHORT_ROWS * (D + 4));
    float(*const s_l)[SHORT_ROWS] = s_m + WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, c = lane >> 4;
    const int H = a.c.kv_heads, P = a.c.page_size, lp = a.c.log2_page;
    const int h = group % H, split = group / H % plan.splits_short;
    const int x = group / H / plan.splits_short;
    int b = x / plan.short_tiles, tile = x % plan.short_tiles;  // (of the sequence)
    if (plan.listed) {
        const int most = plan.short_rows / plan.group;
        const auto tiles = [&](int i) {
            const int n = a.cu_q[i + 1] - a.cu_q[i];
            return n > 0 && n <= most ? (n * plan.group + SHORT_ROWS - 1) / SHORT_ROWS : 0;
        };
        if (plan.short_tiles == 1 ? !find_one(a.s.batch, x, false, tiles, b) : !find_item(a.s.batch, x, false, tiles, b, tile)) return;
    }
    Sequence sq;
    if (!sequence_of(a, b, sq) || sq.n * plan.group > plan.short_rows) return;
    const int row0 = tile * SHORT_ROWS, rows = min(sq.n * plan.group - row0, SHORT_ROWS);
    if (rows <= 0) return;
    const bool mine = n < rows;
    const int tok = (row0 + (mine ? n : 0)) / plan.group, head = h * plan.group + (row0 + (mine ? n : 0)) % plan.group;
    int lo, hi, first_lo, first_hi, last_lo, last_hi;
    seen_range(a, sq, sq.first + tok, lo, hi);
    seen_range(a, sq, sq.first + row0 / plan.group, first_lo, first_hi);
    seen_range(a, sq, sq.first + (row0 + rows - 1) / plan.group, last_lo, last_hi);
    if (!mine) hi = 0;
    // this part's steps of 64 keys: every WAVES-th is this wave's
    const int t_lo = first_lo / TILE, t_hi = (last_hi + TILE - 1) / TILE;
    const int per = max(t_hi - t_lo + plan.splits_short - 1, 0) / plan.splits_short;
    const int begin = t_lo + split * per, end = min(begin + per, t_hi);

    // The channels that lane group c takes in k step s are 8 of its 16 in channels 64 (s / 2) and on (of 32,
    // 8 in the last step, where head_dim is no multiple of 64): a load of 16 codes by all lanes is then
    // 64 whole bytes of each of 16 keys.
    auto channel = [&](int s) { return s / 2 < D / 64 ? 64 * (s / 2) + 16 * c + 8 * (s % 2) : 64 * (D / 64) + 8 * c; };
    // (the first keys are asked for before the row is looked at: each waits for memory once)
    float raw[STEPS][8];
    {
        const int64_t at = (sq.t0 + tok) * a.q.token_stride + (int64_t)head * a.q.head_stride;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) raw[s][j] = load_value<DT>(a.q.p, at + channel(s) + j);
    }
    f32x4 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    Base base;

    const int32_t *table = a.s.tables + b * a.s.table_stride;
    const int64_t page_bytes = (int64_t)P * D;
    const int kg = (lane & 15) >> 2;  // the 16-key group of this lane's rows of K
    // pages of 16-key group g of step t; -1 where there is none to see
    auto page_of = [&](int t, int g) {
        const int key = t * TILE + 16 * g;
        int32_t p = -1;
        if (t < end && key < last_hi) p = table[key >> lp];
        return p >= 0 && p < a.c.num_pages ? p : -1;
    };
    // one step's codes: keys are asked for when the last step's keys have gone into their products, values
    // likewise (with registers for two steps' codes the wave copied a ninth of its instructions)
    uint32_t kc[4][D / 16];
    u32x4 vc[DB];
    auto load_keys = [&](int t, int32_t kp) {
        const uint8_t *p = a.c.k + ((int64_t)max(kp, 0) * H + h) * page_bytes;
        const int at = (t * TILE + 16 * kg) & (P - 1);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint8_t *row = p + (at + 4 * i + (lane & 3)) * D;
#pragma unroll
            for (int j = 0; j < D / 64; j++) {
                const u32x4 w = *reinterpret_cast<const u32x4 *>(row + channel(2 * j));
                kc[i][4 * j] = w[0], kc[i][4 * j + 1] = w[1], kc[i][4 * j + 2] = w[2], kc[i][4 * j + 3] = w[3];
            }
            if constexpr (D % 64 != 0) {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(row + channel(STEPS - 1));
                kc[i][2 * STEPS - 2] = w[0], kc[i][2 * STEPS - 1] = w[1];
            }
        }
    };
    auto load_values = [&](int t, int32_t vp) {
        const uint8_t *p = a.c.v + ((int64_t)max(vp, 0) * H + h) * page_bytes + n * P + ((t * TILE + 16 * c) & (P - 1));
#pragma unroll
        for (int i = 0; i < DB; i++) vc[i] = *reinterpret_cast<const u32x4 *>(p + i * 16 * P);
    };
    auto load_scales = [&](int32_t vp, float &k, float &v) {
        const int64_t vh = (int64_t)max(vp, 0) * H + h;
        k = a.c.ks[vh];
        v = vp >= 0 ? a.c.vs[vh] : 0.f;
    };

    int t = begin + wave;
    int32_t vp = page_of(t, c), kp = page_of(t, kg);
    int32_t vp_next = page_of(t + WAVES, c), kp_next = page_of(t + WAVES, kg);
    float ks = 0.f, vs = 0.f;
    if (t < end) {
        load_keys(t, kp);
        load_scales(vp, ks, vs);
        load_values(t, vp);
    }
    // the row's parts or digits, and the factor of its logits (in powers of two)
    half8 q[DIGITS ? 1 : STEPS][NS];
    uint32_t qd[4][DIGITS ? D / 16 : 1];
    float factor;
    {
        uint32_t most = 0;  // (as whole numbers: what is not finite is the largest)
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(fabsf(raw[s][j])));
        most = max(most, (uint32_t)__shfl_xor((int)most, 16));
        most = max(most, (uint32_t)__shfl_xor((int)most, 32));
        constexpr int BITS = DIGITS ? 31 : 15;
        int e = row_exponent(__uint_as_float(most));
        if (DIGITS && ldexpf(__uint_as_float(most), BITS - e) > MOST_DIGITS) e++;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
#pragma unroll
            for (int j = 0; j < 8; j++) raw[s][j] = copysignf(1.f, a.scale) * ldexpf(raw[s][j], BITS - e);
            if constexpr (DIGITS) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    uint32_t d[4];
                    digits4(raw[s] + 4 * j, d);
#pragma unroll
                    for (int i = 0; i < 4; i++) qd[i][2 * s + j] = d[i];
                }
            } else {
                parts8<NS>(raw[s], q[s]);
            }
        }
        factor = ldexpf(fabsf(a.scale) * 1.44269504088896340736f, e - (DIGITS ? BITS - 8 : BITS));  // (their products count in 2^8)
        // digits cannot say so, and one f16 part would leave a row of which all logits are -infinity as one that sees nothing
        if (most >= 0x7f800000u) factor = __uint_as_float(0x7fc00000u);
    }
    // (the older wave of a SIMD goes first where both could, and would be done long before the other)
    if (wave >= 4) __builtin_amdgcn_s_setprio(1);
    for (; t < end; t += WAVES) {
        const bool more = t + WAVES < end;
        const int32_t vp_far = page_of(t + 2 * WAVES, c), kp_far = page_of(t + 2 * WAVES, kg);

        const int key = t * TILE;
        float x[16];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DIGITS) {
                i32x4 s[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
                for (int u = 0; u < 4; u++) {
#pragma unroll
                    for (int j = 0; j < D / 64; j++)
                        s[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                            (i32x4){(int)kc[i][4 * j], (int)kc[i][4 * j + 1], (int)kc[i][4 * j + 2], (int)kc[i][4 * j + 3]},
                            (i32x4){(int)qd[u][4 * j], (int)qd[u][4 * j + 1], (int)qd[u][4 * j + 2], (int)qd[u][4 * j + 3]}, s[u], 0, 0, 0);
                    if constexpr (D % 64 != 0)  // (the last 32 channels, and zeros)
                        s[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8((i32x4){(int)kc[i][D / 16 - 2], (int)kc[i][D / 16 - 1], 0, 0},
                                                                    (i32x4){(int)qd[u][D / 16 - 2], (int)qd[u][D / 16 - 1], 0, 0}, s[u], 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < 4; j++)  // 2^-8 of it, each half a whole number below 2^31
                    x[4 * i + j] = fmaf((float)(256 * s[3][j] + s[2][j]), 256.f, (float)(256 * s[1][j] + s[0][j]) * 0x1p-8f);
            } else {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < STEPS; j++) {
                    const half8 k8 = codes8<KIND>(kc[i][2 * j], kc[i][2 * j + 1]);
#pragma unroll
                    for (int u = NS - 1; u >= 0; u--) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, q[j][u], s, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) x[4 * i + j] = s[j];
            }
        }
        float ks_next = 0.f, vs_next = 0.f;
        if (more) {
            load_keys(t + WAVES, kp_next);
            load_scales(vp_next, ks_next, vs_next);
        }
        float vmax = fmaxf(vs, __shfl_xor(vs, 16));
        vmax = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(fmaxf(vmax, __shfl_xor(vmax, 32)))));
        if (vmax > base.r) {
            const float row_l = fmaxf(l, __shfl_xor(l, 16));
            const float g = base.grow(scale_ceiling(vmax), l, fmaxf(row_l, __shfl_xor(row_l, 32)));
#pragma unroll
            for (int i = 0; i < DB; i++) o[i] *= g;
        }
        float f = ks * factor, lv = scale_log(vs, base.inv_r);  // f >= 0: the largest product has the largest logit
        if (key < last_lo || key + TILE > first_hi || __any(vp < 0)) {
            // some row does not see some of these keys, or they are not there
            const int from = lo - (key + 16 * c), to = vp >= 0 ? hi - (key + 16 * c) : 0;
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = seen_or_not(x[j], j, from, to);
            f = not_zero(f);
            if (max(from, 0) >= min(to, 16)) f = 1.f, lv = 0.f;  // none of them, so neither their scales
            const int keep = vp >= 0 ? min(max(sq.len - (key + 16 * c), 0), 16) : 0;
#pragma unroll
            for (int i = 0; i < DB; i++) vc[i] = keep_bytes(vc[i], keep);
        }
        float top = larger(x[0], x[1]);
#pragma unroll
        for (int j = 2; j < 16; j++) top = fmaxf(top, x[j]);
        top = fmaf(top, f, lv);  // of this lane's keys; the row's only where the base has to move
        if (__any(top > base.b + LAZY_LOG2)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float g = base.move(top);
            l *= g;
#pragma unroll
            for (int i = 0; i < DB; i++) o[i] *= g;
        }
        const float at = base_of(base.b) - WEIGHT_LOG2 - lv;
        float w[16], sum = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            w[j] = exp2_fast(fmaf(x[j], f, -at));
            sum += w[j];
        }
        l = fmaf(sum, exp2_fast(-lv), l);
        half8 p[2][NW];
        parts8<NW>(w, p[0]);
        parts8<NW>(w + 8, p[1]);
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const half8 v8 = codes8<KIND>(vc[i][2 * u], vc[i][2 * u + 1]);
#pragma unroll
                for (int z = NW - 1; z >= 0; z--) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, p[u][z], o[i], 0, 0, 0);
            }
        if (more) load_values(t + WAVES, vp_next);
        ks = ks_next, vs = vs_next;
        vp = vp_next, kp = kp_next;
        vp_next = vp_far, kp_next = kp_far;
    }

    // the waves' parts, then theirs joined: channel by channel
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (apart from r: their quotient can be subnormal)
    settle(base.b, l);
#pragma unroll
    for (int i = 0; i < DB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s_o[wave][n][16 * i + 4 * c + j] = l == 0.f ? 0.f : o[i][j] * inv * base.r;
    if (c == 0) s_m[wave][n] = base.b, s_l[wave][n] = l;
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * WAVES) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        float top = -INFINITY, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, s_m[w][row]);
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float f = part_weight(s_m[w][row], s_l[w][row], top);
            sum += f;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = fmaf(f, s_o[w][row][d + j], v[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = sum == 0.f ? 0.f : v[j] / sum;
        const int tok = (row0 + row) / plan.group, head = h * plan.group + (row0 + row) % plan.group;
        if (plan.splits_short == 1) {
            store_values4<DT>(a.out, ((int64_t)(sq.t0 + tok) * a.q_heads + head) * D + d, v);
        } else {
            const int64_t unit = plan.short_per ? b * plan.short_per + tok : sq.t0 + tok, at = (split * plan.short_tokens + unit) * a.q_heads + head;
            *reinterpret_cast<f32x4 *>(plan.part + at * D + d) = f32x4{v[0], v[1], v[2], v[3]};
            if (d == 0) plan.stat[2 * at] = top, plan.stat[2 * at + 1] = sum;
        }
    }
}

// Waves of a workgroup where all sequences are short: as many as the registers allow on a CU, so
// that most batches need no parts and no join.
template <int D>
constexpr int SHORT_WAVES = D <= 128 ? 8 : 4;

template <int D, int KIND, int DT>
__global__ __launch_bounds__(64 * SHORT_WAVES<D>, D <= 128 ? 2 : 1) void k_attn_short(KvAttention a, AttnPlan plan) {
    extern __shared__ __align__(16) float lds_f[];
    attn_short<D, KIND, DT, SHORT_WAVES<D>>(a, plan, blockIdx.x, lds_f);
}

// ---------------------------------------------------------------------------
// Long form: query rows of one kv head (row i * group + head: neighbouring tokens see nearly the
// same keys), 32 for each wave.  Long prompts are bound by the matrix cores and by the vector unit's weights
// (seven instructions each), which hardly run at once within a wave; calls of few workgroups, or of unlike ones, by
// the longest of them, by barriers and by waves without rows.  64 keys at a
// time are turned into f16 once for all waves and kept in LDS, the next steps' codes on their
// way from memory meanwhile.  32x32x16 products; rows of K lie in LDS in the order in which lane
// (half, n) then holds keys 16 u + 8 half + j of its row n, what the products with V take.
// LDS rows are an odd number of 16-byte chunks long, so that eight lanes' reads of one column
// use all banks.
//
// Pages and scales of up to 256 steps are looked up at once, by all threads, and kept in LDS: offsets
// of the pages' codes, key scales, value scales as they enter the exponential.  (Looked up step by
// step they took a quarter of a step's time, most of it address arithmetic.)
//
// Up to 128 channels the registers allow two waves on a SIMD, and one's products run while the
// other forms weights.  Above that there is one, and four in a workgroup.  In either case the
// weights of 16 keys are formed between the products of the 16 before.
//
// A prompt of 8000 tokens in bf16, 32 heads of 128 channels, window 5000, 450.6 GFLOP: 463 to 479 us,
// 0.94 to 0.97 PFLOP/s (a large library product: 1.14); the matrix cores are busy in 41 % of the cycles, the vector
// unit in 47 %, at 2.0 of 2.4 GHz: the power limit, as far as the clock says.  Four chunks of 512 over contexts of 1500
// in f32, 38.7 GFLOP and twice the products: 98 us, units busy in 31 and 26 %.  220 rows a head over 1500 states of 64
// channels in f16: 44 us on 160 CUs, where 4 to 7 of 8 waves have rows and the units are busy in 18 and 34 %.  Measured and no
// better: steps of 128 keys (64 channels: -3 %, causal prompts +2 %), codes two steps ahead, four waves a workgroup
// (618 us for the prompt), three buffers with the waves half a step apart (665), sums by dot products.
// ---------------------------------------------------------------------------
constexpr int WAVE_ROWS = 32;
template <int D>
constexpr int LONG_WAVES = D <= 128 ? 8 : 4;
constexpr int TABLE_STEPS = 256, GROUPS = TILE / 16;  // steps looked up at once; groups of 16 keys in a step

template <int D>
constexpr int buffer_halves() { return TILE * (D + 8) + D * (TILE + 8); }  // f16 of one step's K and V
template <int D>
constexpr size_t long_lds() { return 2 * sizeof(_Float16) * buffer_halves<D>() + TABLE_STEPS * GROUPS * (sizeof(uint64_t) + 2 * sizeof(float)); }

// group: its place among the form's workgroups (tiles * kv heads * parts); lds: long_lds bytes
template <int D, int KIND, int DT>
__device__ __forceinline__ void attn_long(const KvAttention &a, const AttnPlan &plan, int group, _Float16 *lds) {
    constexpr int NS = QUERY_PARTS<DT>, NW = WEIGHT_PARTS<DT>, WAVES = LONG_WAVES<D>, ROWS = WAVE_ROWS * WAVES, THREADS = 64 * WAVES;
    constexpr int STEPS = D / 16, DB = D / 32;
    constexpr int KROW = D + 8, VROW = TILE + 8;
    constexpr int CHUNKS = TILE * D / 16, PER = (CHUNKS + THREADS - 1) / THREADS;  // 16-code chunks, of K and of V
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, hf = lane >> 5;
    const int H = a.c.kv_heads, P = a.c.page_size, lp = a.c.log2_page;
    // the tiles with most keys (a sequence's last) first
    const int h = group % H, split = group / H % plan.splits_long;
    int b, tile;  // (of the sequence)
    if (plan.listed) {
        const int least = plan.short_rows / plan.group, most = plan.tiles_per ? plan.tiles_per : plan.tiles, x = group / H / plan.splits_long;
        const auto new_tokens = [&](int i) { return a.cu_q[i + 1] - a.cu_q[i]; };
        if (most == 1) {
            tile = 0;
            if (!find_one(a.s.batch, x, true, [&](int i) { return new_tokens(i) > least; }, b)) return;
        } else {
            const auto tiles = [&](int i) {
                const int n = new_tokens(i);
                return n > least ? (int)min(((int64_t)n * plan.group + ROWS - 1) / ROWS, (int64_t)most) : 0;
            };
            if (!find_item(a.s.batch, x, true, tiles, b, tile)) return;
        }
    } else {
        tile = plan.tiles - 1 - group / H / plan.splits_long;
        b = plan.tiles_per ? tile / plan.tiles_per
                           : find_sequence(a.s.batch, tile, [&](int i) { return (int64_t)a.cu_q[i] * plan.group / ROWS + i; });
        tile -= plan.tiles_per ? b * plan.tiles_per : (int)((int64_t)a.cu_q[b] * plan.group / ROWS) + b;
    }
    Sequence sq;
    if (!sequence_of(a, b, sq) || sq.n * plan.group <= plan.short_rows) return;
    const int rows = sq.n * plan.group;
    if (tile < 0 || tile >= (rows + ROWS - 1) / ROWS) return;
    const int row0 = tile * ROWS;
    const int row = row0 + WAVE_ROWS * wave + n;
    const bool mine = row < rows;
    const int tok = (mine ? row : rows - 1) / plan.group, head = h * plan.group + (mine ? row : rows - 1) % plan.group;
    int lo, hi;  // keys that this lane's row sees
    seen_range(a, sq, sq.first + tok, lo, hi);
    int begin, end;  // steps of this part
    {
        int first_lo, first_hi, last_lo, last_hi;
        seen_range(a, sq, sq.first + row0 / plan.group, first_lo, first_hi);
        seen_range(a, sq, sq.first + (min(row0 + ROWS, rows) - 1) / plan.group, last_lo, last_hi);
        const int t_lo = first_lo / TILE, t_hi = (last_hi + TILE - 1) / TILE;
        const int per = max(t_hi - t_lo + plan.splits_long - 1, 0) / plan.splits_long;
        begin = t_lo + split * per, end = min(begin + per, t_hi);
    }
    int see_lo, see_hi, all_lo, all_hi;  // steps of which any row of this wave sees a key; of which every row sees all
    {
        const int w0 = row0 + WAVE_ROWS * wave, w1 = min(w0 + WAVE_ROWS, rows) - 1;
        int first_lo, first_hi, last_lo, last_hi;
        seen_range(a, sq, sq.first + min(w0, rows - 1) / plan.group, first_lo, first_hi);
        seen_range(a, sq, sq.first + w1 / plan.group, last_lo, last_hi);
        see_lo = first_lo / TILE, see_hi = w0 < rows ? min((last_hi + TILE - 1) / TILE, end) : 0;
        all_lo = (last_lo + TILE - 1) / TILE, all_hi = first_hi / TILE;
    }
    auto visible = [&](int t) { return t >= see_lo && t < see_hi; };

    half8 q[STEPS][NS];
    float factor;
    {
        const int64_t at = (sq.t0 + tok) * a.q.token_stride + (int64_t)head * a.q.head_stride + 8 * hf;
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < STEPS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(load_value<DT>(a.q.p, at + 16 * i + j)));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        const int e = row_exponent(amax);
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = copysignf(1.f, a.scale) * ldexpf(load_value<DT>(a.q.p, at + 16 * i + j), 15 - e);
            parts8<NS>(v, q[i]);
        }
        factor = ldexpf(fabsf(a.scale) * 1.44269504088896340736f, e - 15);
        if (amax == INFINITY) factor = __uint_as_float(0x7fc00000u);  // (as in attn_short; NaN is in the products)
    }

    f32x16 o[DB], s[2];
#pragma unroll
    for (int i = 0; i < DB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[i][j] = 0.f;
    float l = 0.f;
    Base base;

    // ---- the steps' pages and scales
    _Float16 *const buffers = lds;
    uint64_t *const s_at = reinterpret_cast<uint64_t *>(lds + 2 * buffer_halves<D>());  // bytes from the cache's start to the group's page
    float *const s_k = reinterpret_cast<float *>(s_at + TABLE_STEPS * GROUPS);          // key scales, -1: the group is not there
    float *const s_lv = s_k + TABLE_STEPS * GROUPS;  // scale_log of value scales
    __shared__ float s_max[WAVES];
    __shared__ int s_missing[WAVES];
    bool missing = false;  // whether a group that a row could see is not there
    const int32_t *const table = a.s.tables + b * a.s.table_stride;
    const int seen_end = min(end * TILE, sq.len);
    // the entries of steps c0 .. c1 - 1; grown: whether r grew, and the outputs have to be multiplied by `by`
    auto look_up = [&](int c0, int c1, bool &grown, float &by) {
        const int n = (c1 - c0) * GROUPS;
        float vmax = 0.f;
        bool lacks = false;
        for (int i = tid; i < n; i += THREADS) {
            const int key = c0 * TILE + 16 * i;
            const int page = key < seen_end ? table[key >> lp] : -1;
            const bool there = page >= 0 && page < a.c.num_pages;
            const int64_t at = there ? (int64_t)page * H + h : 0;
            const float v = there ? a.c.vs[at] : 0.f;
            s_at[i] = at * (uint64_t)(P * D);
            s_k[i] = there ? a.c.ks[at] : -1.f;
            s_lv[i] = v;
            vmax = fmaxf(vmax, v);
            lacks |= key < seen_end && !there;
        }
#pragma unroll
        for (int d = 32; d; d /= 2) vmax = fmaxf(vmax, __shfl_xor(vmax, d));
        const bool any = __any(lacks);
        if (lane == 0) s_max[wave] = vmax, s_missing[wave] = any;
        __syncthreads();
        missing = false;
#pragma unroll
        for (int i = 0; i < WAVES; i++) vmax = fmaxf(vmax, s_max[i]), missing |= s_missing[i] != 0;
        missing = __any(missing);
        grown = vmax > base.r;  // (the same in every thread)
        if (grown) by = base.grow(scale_ceiling(vmax), l, fmaxf(l, __shfl_xor(l, 32)));
        for (int i = tid; i < n; i += THREADS) s_lv[i] = scale_log(s_lv[i], base.inv_r);
        __syncthreads();
    };

    // ---- codes on their way.  A thread has the same chunks of 16 codes in every step: of K key `kt`
    // of the step, channels kd and on; of V channel `vd`, keys 16 vg and on.
    struct Chunk {
        int kt, kd, vg, vd;
        bool on;
    };
    auto chunk = [&](int i) {
        const int id = tid + THREADS * i;
        return Chunk{id / (D / 16), id % (D / 16) * 16, id & 3, id >> 2, CHUNKS % THREADS == 0 || id < CHUNKS};
    };
    u32x4 kc[PER], vc[PER];
    uint64_t k_at[PER], v_at[PER];  // of the step to load next
    auto read_places = [&](int i) {  // entry i of the table
#pragma unroll
        for (int j = 0; j < PER; j++) {
            k_at[j] = s_at[GROUPS * i + (chunk(j).kt >> 4 & 3)];
            v_at[j] = s_at[GROUPS * i + chunk(j).vg];
        }
    };
    auto load = [&](int t) {
        const int in_page = t * TILE & (P - 1);  // (pages of 128: the step is one half of one)
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const Chunk c = chunk(j);
            if (c.on) {
                kc[j] = *reinterpret_cast<const u32x4 *>(a.c.k + k_at[j] + ((in_page + (c.kt & (P - 1))) * D + c.kd));
                vc[j] = *reinterpret_cast<const u32x4 *>(a.c.v + v_at[j] + (c.vd * P + in_page + (16 * c.vg & (P - 1))));
            }
        }
    };
    // codes -> f16 in buffer `buf`.  Values behind the sequence's end, or of no page, as zeros: their
    // weights are 0, but a code can be NaN.
    auto stage = [&](int t, int i, int buf) {
        _Float16 *const kb = buffers + buf * buffer_halves<D>(), *const vb = kb + TILE * KROW;
        if (missing || (t + 1) * TILE > sq.len) {
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int vg = chunk(j).vg;
                vc[j] = keep_bytes(vc[j], s_k[GROUPS * i + vg] < 0.f ? 0 : min(max(sq.len - (t * TILE + 16 * vg), 0), 16));
            }
        }
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const Chunk c = chunk(j);
            if (c.on) {
                // key 32 b + 16 a1 + 8 half + 4 a0 + j is row 32 b + 16 a1 + 8 a0 + 4 half + j
                const int kr = (c.kt & 0x33) | (c.kt & 8) >> 1 | (c.kt & 4) << 1;
                half8 *const ko = reinterpret_cast<half8 *>(kb + kr * KROW + c.kd);
                ko[0] = codes8<KIND>(kc[j][0], kc[j][1]);
                ko[1] = codes8<KIND>(kc[j][2], kc[j][3]);
                half8 *const vo = reinterpret_cast<half8 *>(vb + c.vd * VROW + 16 * c.vg);
                vo[0] = codes8<KIND>(vc[j][0], vc[j][1]);
                vo[1] = codes8<KIND>(vc[j][2], vc[j][3]);
            }
        }
    };

    // ---- products.  Operands in groups of up to four, the next group read before the products of
    // the last: left to itself the compiler reads each right before its product and waits for it.
    half8 fr[2][4], p[4][NW];
    auto read_keys = [&](int g, const _Float16 *kb) {  // k dimensions 2 g and 2 g + 1, both blocks of 32 keys
#pragma unroll
        for (int z = 0; z < 4; z++) fr[g & 1][z] = *reinterpret_cast<const half8 *>(kb + (32 * (z & 1) + n) * KROW + 16 * (2 * g + z / 2) + 8 * hf);
    };
    auto key_products = [&](const _Float16 *kb) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[i][j] = 0.f;
        read_keys(0, kb);
#pragma unroll
        for (int g = 0; g < STEPS / 2; g++) {
            if (g + 1 < STEPS / 2) read_keys(g + 1, kb);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int z = 0; z < 4; z++)
#pragma unroll
                for (int u = NS - 1; u >= 0; u--)
                    s[z & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[g & 1][z], q[2 * g + z / 2][u], s[z & 1], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr int VG = DB <= 4 ? DB : DB / 2, VGROUPS = 4 * DB / VG;  // channel blocks in a group of operands of V
    auto read_values = [&](int g, const _Float16 *vb) {
#pragma unroll
        for (int i = 0; i < VG; i++)
            fr[g & 1][i] = *reinterpret_cast<const half8 *>(vb + (32 * (g % (DB / VG) * VG + i) + n) * VROW + 16 * (g / (DB / VG)) + 8 * hf);
    };
    auto value_products = [&](int g) {
#pragma unroll
        for (int z = NW - 1; z >= 0; z--)
#pragma unroll
            for (int i = 0; i < VG; i++) {
                f32x16 &to = o[g % (DB / VG) * VG + i];
                to = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[g & 1][i], p[g / (DB / VG)][z], to, 0, 0, 0);
            }
    };

    // ---- weights.  s[i][j] is key 16 u + 8 hf + 4 (j / 4 % 2) + j % 4 of the step, u = 2 i + j / 8
    auto scale_outputs = [&](float by) {
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[i][j] *= by;
    };
    float f[4], lv[4];
    auto start_weights = [&](int t, int i) {  // entry i of the table
        const f32x4 k4 = *reinterpret_cast<const f32x4 *>(s_k + GROUPS * i), lv4 = *reinterpret_cast<const f32x4 *>(s_lv + GROUPS * i);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            f[u] = k4[u] * factor;  // not negative where a key is seen: the largest product has the largest logit
            lv[u] = lv4[u];
        }
        if (missing || t < all_lo || t >= all_hi) {
            // some row does not see some of these keys, or they are not there
            const int from = lo - (t * TILE + 8 * hf), to = hi - (t * TILE + 8 * hf);
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int a0 = max(from - 16 * u, 0), a1 = k4[u] < 0.f ? 0 : min(to - 16 * u, 8);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = s[u / 2][8 * (u % 2) + j];
                    s[u / 2][8 * (u % 2) + j] = seen_or_not(x, j, a0, a1);
                }
                f[u] = not_zero(f[u]);
                if (a0 >= a1) f[u] = 1.f, lv[u] = 0.f;  // none of the group, so neither its scales
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float x = larger(s[u / 2][8 * (u % 2)], s[u / 2][8 * (u % 2) + 1]);
#pragma unroll
            for (int j = 2; j < 8; j++) x = fmaxf(x, s[u / 2][8 * (u % 2) + j]);
            top = fmaxf(top, fmaf(x, f[u], lv[u]));
        }
        if (__any(top > base.b + LAZY_LOG2)) {  // (this lane's keys; the row's only where the base has to move)
            const float g = base.move(fmaxf(top, __shfl_xor(top, 32)));
            l *= g;
            scale_outputs(g);
        }
    };
    auto weigh = [&](int u) {
        const float at = base_of(base.b) - WEIGHT_LOG2 - lv[u];
        float w[8], sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            w[j] = exp2_fast(fmaf(s[u / 2][8 * (u % 2) + j], f[u], -at));
            sum += w[j];
        }
        l = fmaf(sum, exp2_fast(-lv[u]), l);
        parts8<NW>(w, p[u]);
    };

    for (int c0 = begin; c0 < end; c0 += TABLE_STEPS) {
        const int n = min(end - c0, TABLE_STEPS);
        bool grown;
        float by;
        look_up(c0, c0 + n, grown, by);
        if (grown) scale_outputs(by);
        read_places(0);
        load(c0);
        read_places(min(1, n - 1));
        stage(c0, 0, 0);
        __syncthreads();
        for (int i = 0; i < n; i++) {
            const int t = c0 + i, buf = i & 1;
            if (i + 1 < n) load(t + 1);
            if (visible(t)) {
                const _Float16 *const kb = buffers + buf * buffer_halves<D>(), *const vb = kb + TILE * KROW;
                // (a wave's products go before the other's weights where both could go)
                __builtin_amdgcn_s_setprio(1);
                key_products(kb);
                __builtin_amdgcn_s_setprio(0);
                start_weights(t, i);
                read_values(0, vb);
                weigh(0);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int g = 0; g < VGROUPS; g++) {
                    if (g + 1 < VGROUPS) read_values(g + 1, vb);
                    __builtin_amdgcn_sched_barrier(0);
                    value_products(g);
                    const int u = g / (DB / VG) + 1;
                    if (g % (DB / VG) == 0 && u < 4) {
                        weigh(u);
                        constexpr int MFMA = 0x8, VALU = 0x2, TRANS = 0x400;
#pragma unroll
                        for (int j = 0; j < VG * NW; j++) {
                            __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(VALU | TRANS, 32 / (VG * NW) + 1, 0);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(0);
            }
            if (i + 1 < n) {
                stage(t + 1, i + 1, buf ^ 1);
                read_places(min(i + 2, n - 1));
            }
            __syncthreads();
        }
    }

    l += __shfl_xor(l, 32);
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (apart from r: their quotient can be subnormal)
    if (!mine) return;
    const int64_t out = (sq.t0 + tok) * a.q_heads + head, at = plan.long_row + split * a.num_q * a.q_heads + out;
    if (plan.splits_long > 1) {
        settle(base.b, l);
        if (hf == 0) plan.stat[2 * at] = base.b, plan.stat[2 * at + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < DB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float v[4];
#pragma unroll
            for (int z = 0; z < 4; z++) v[z] = l == 0.f ? 0.f : o[i][4 * j + z] * inv * base.r;
            const int d = 32 * i + 8 * j + 4 * hf;
            if (plan.splits_long == 1) store_values4<DT>(a.out, out * D + d, v);
            else *reinterpret_cast<f32x4 *>(plan.part + at * D + d) = f32x4{v[0], v[1], v[2], v[3]};
        }
}

// Both forms in one launch, each sequence in its own: short_groups workgroups of the short form,
// which are the first to start (a long context's single token takes longest), then the long form's.
template <int D, int KIND, int DT>
__global__ __launch_bounds__(64 * LONG_WAVES<D>, D <= 128 ? 2 : 1) void k_attn_mixed(KvAttention a, AttnPlan plan, int short_groups) {
    extern __shared__ __align__(16) _Float16 lds_h[];
    if ((int)blockIdx.x < short_groups) attn_short<D, KIND, DT, LONG_WAVES<D>>(a, plan, blockIdx.x, reinterpret_cast<float *>(lds_h));
    else attn_long<D, KIND, DT>(a, plan, blockIdx.x - short_groups, lds_h);
}

// The join of a row's parts, D / 4 threads a row.  Few rows: a workgroup for one row, whose groups take
// every JOIN_GROUPS-th part and are added in order.  Many: a row for each group of threads.  Bound by
// latency: a row's workgroup asks for maxima, parts and the row's bounds at once (one after the
// other 8000 keys in 62 parts took 15.7 us, now 11.9).  From the call's time: 32 rows of 15 parts 16.8 us
// with a workgroup a row, 18.5 with a group of threads; 128 rows of 7 parts 16.8 and 18.0; 3200 rows of 15
// parts 47.8 and 46.0; 16384 rows of 4 parts 67.4 and 52.
// The rows are the short form's, if it cut its sequences, and then the long form's, if that did.
constexpr int JOIN_THREADS = 256, JOIN_ROWS = 1024;  // rows up to which each has a workgroup
template <int D>
constexpr int JOIN_GROUPS = JOIN_THREADS / (D / 4);

// a row of the parts: whose it is, without the sequence's bounds
struct PartRow {
    bool is_short;
    int splits;
    int64_t row, all, at;  // (token, head) in its form's order; rows of one part; its place in the first part
};
__device__ __forceinline__ PartRow part_row(const KvAttention &a, const AttnPlan &plan, int64_t id) {
    const int64_t short_rows = plan.splits_short > 1 ? plan.short_tokens * a.q_heads : 0;
    PartRow r;
    r.is_short = id < short_rows;
    r.splits = r.is_short ? plan.splits_short : plan.splits_long;
    r.row = r.is_short ? id : id - short_rows;
    r.all = r.is_short ? short_rows : a.num_q * a.q_heads;
    r.at = r.row + (r.is_short ? 0 : plan.long_row);
    return r;
}
// the batch's token t of a row, given sequence b that begins at or before t; false where no sequence has it in this
// form, or where it lies behind the tiles that the bound on new tokens gives (its parts are nobody's)
template <int D, class Find>
__device__ __forceinline__ bool part_token(const KvAttention &a, const AttnPlan &plan, const PartRow &r, Find find, int64_t &t) {
    t = r.row / a.q_heads;
    const bool own = r.is_short && plan.short_per;
    const int b = own ? (int)(t / plan.short_per) : find(t);
    Sequence sq;
    if (!sequence_of(a, b, sq)) return false;
    if (own) t += sq.t0 - (int64_t)b * plan.short_per;
    if (!r.is_short && plan.tiles_per) {
        const int64_t row = (t - sq.t0) * plan.group + r.row % a.q_heads % plan.group;
        if (row >= (int64_t)plan.tiles_per * WAVE_ROWS * LONG_WAVES<D>) return false;
    }
    return t >= sq.t0 && t < sq.t0 + sq.n && (sq.n * plan.group <= plan.short_rows) == r.is_short;
}

template <int D, int DT>
__global__ __launch_bounds__(JOIN_THREADS) void k_attn_join_row(KvAttention a, AttnPlan plan) {
    constexpr int G = JOIN_GROUPS<D>, AHEAD = 8;
    __shared__ f32x4 s_v[G][D / 4];
    __shared__ float s_f[JOIN_THREADS], s_top[JOIN_THREADS / 64], s_sum[JOIN_THREADS / 64];
    const int tid = threadIdx.x, wave = tid >> 6, g = tid / (D / 4), d = tid % (D / 4) * 4;
    const PartRow r = part_row(a, plan, blockIdx.x);
    // everything is asked for before the row's sequence is known
    float m = -INFINITY, l = 0.f;
    if (tid < r.splits) {
        const float *const stat = plan.stat + 2 * (r.at + tid * r.all);
        m = stat[0], l = stat[1];
    }
    const float *const part = plan.part + r.at * D + d;
    f32x4 x[AHEAD];
#pragma unroll
    for (int z = 0; z < AHEAD; z++)
        x[z] = g < G && g + z * G < r.splits ? *reinterpret_cast<const f32x4 *>(part + (g + z * G) * r.all * D) : f32x4{0.f, 0.f, 0.f, 0.f};
    int64_t t;
    if (!part_token<D>(a, plan, r, [&](int64_t at) { return find_sequence(a.s.batch, at, [&](int i) { return (int64_t)a.cu_q[i]; }); }, t)) return;
    float top = m;
#pragma unroll
    for (int i = 32; i; i /= 2) top = fmaxf(top, __shfl_xor(top, i));
    if ((tid & 63) == 0) s_top[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < JOIN_THREADS / 64; i++) top = fmaxf(top, s_top[i]);
    const float f = part_weight(m, l, top);
    s_f[tid] = f;
    float sum = f;
#pragma unroll
    for (int i = 32; i; i /= 2) sum += __shfl_xor(sum, i);
    if ((tid & 63) == 0) s_sum[wave] = sum;
    __syncthreads();
    f32x4 v = {0.f, 0.f, 0.f, 0.f};  // (a part that saw nothing is zero)
    if (g < G) {
#pragma unroll
        for (int z = 0; z < AHEAD; z++)
            if (g + z * G < r.splits) v += s_f[g + z * G] * x[z];
        for (int i = g + AHEAD * G; i < r.splits; i += G) v += s_f[i] * *reinterpret_cast<const f32x4 *>(part + i * r.all * D);
        s_v[g][d / 4] = v;
    }
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int i = 1; i < G; i++) v += s_v[i][d / 4];
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < JOIN_THREADS / 64; i++) sum += s_sum[i];
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = sum == 0.f ? 0.f : v[j] / sum;
    store_values4<DT>(a.out, (t * a.q_heads + r.row % a.q_heads) * D + d, o);
}

template <int D, int DT>
__global__ __launch_bounds__(JOIN_THREADS) void k_attn_join(KvAttention a, AttnPlan plan, int64_t rows) {
    constexpr int G = JOIN_GROUPS<D>;
    const int g = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const int64_t id = (int64_t)blockIdx.x * G + g;
    if (g >= G || id >= rows) return;
    const PartRow r = part_row(a, plan, id);
    int64_t t;
    const auto find = [&](int64_t at) {
        int b = 0;
        for (int n = a.s.batch; n > 1;) {  // the last sequence that begins at or before the token
            const int half = n / 2;
            const bool up = a.cu_q[b + half] <= at;
            b += up ? half : 0;
            n = up ? n - half : half;
        }
        return b;
    };
    if (!part_token<D>(a, plan, r, find, t)) return;
    const float *const stat = plan.stat + 2 * r.at;
    const float *const part = plan.part + r.at * D + d;
    float top = -INFINITY;
#pragma unroll 8
    for (int i = 0; i < r.splits; i++) top = fmaxf(top, stat[2 * i * r.all]);
    float sum = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < r.splits; i++) {
        const float f = part_weight(stat[2 * i * r.all], stat[2 * i * r.all + 1], top);
        sum += f;
        v += f * *reinterpret_cast<const f32x4 *>(part + i * r.all * D);  // (a part that saw nothing is zero)
    }
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = sum == 0.f ? 0.f : v[j] / sum;
    store_values4<DT>(a.out, (t * a.q_heads + r.row % a.q_heads) * D + d, o);
}

template <int D, int KIND, int DT>
hipError_t launch_typed(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st) {
    const int short_groups = any_short ? plan.splits_short * a.c.kv_heads * plan.short_groups : 0;
    const auto launch = [&](auto k, int groups, int threads, size_t lds, auto... more) {
        if (lds > 65536) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        k<<<dim3((unsigned)groups), threads, lds, st>>>(a, plan, more...);
        return hipGetLastError();
    };
    hipError_t e = hipSuccess;
    if (any_long)
        e = launch(k_attn_mixed<D, KIND, DT>, short_groups + plan.tiles * a.c.kv_heads * plan.splits_long, 64 * LONG_WAVES<D>,
                   std::max(long_lds<D>(), short_lds<D, LONG_WAVES<D>>()), short_groups);
    else if (any_short)
        e = launch(k_attn_short<D, KIND, DT>, short_groups, 64 * SHORT_WAVES<D>, short_lds<D, SHORT_WAVES<D>>());
    if (e != hipSuccess) return e;
    if (plan.splits_short == 1 && plan.splits_long == 1) return hipSuccess;
    const int64_t rows = (plan.splits_short > 1 ? plan.short_tokens * a.q_heads : 0) + (plan.splits_long > 1 ? a.num_q * a.q_heads : 0);
    if (rows <= JOIN_ROWS) k_attn_join_row<D, DT><<<dim3((unsigned)rows), JOIN_THREADS, 0, st>>>(a, plan);
    else k_attn_join<D, DT><<<dim3((unsigned)((rows + JOIN_GROUPS<D> - 1) / JOIN_GROUPS<D>)), JOIN_THREADS, 0, st>>>(a, plan, rows);
    return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st) {
    const bool i8 = a.c.kind == KV_INT8;
    switch (a.dtype) {
        case DT_F32:
            return i8 ? launch_typed<D, KV_INT8, DT_F32>(a, plan, any_short, any_long, st) : launch_typed<D, KV_E4M3, DT_F32>(a, plan, any_short, any_long, st);
        case DT_F16:
            return i8 ? launch_typed<D, KV_INT8, DT_F16>(a, plan, any_short, any_long, st) : launch_typed<D, KV_E4M3, DT_F16>(a, plan, any_short, any_long, st);
        default:
            return i8 ? launch_typed<D, KV_INT8, DT_BF16>(a, plan, any_short, any_long, st) : launch_typed<D, KV_E4M3, DT_BF16>(a, plan, any_short, any_long, st);
    }
}

}  // namespace attn

// one translation unit per head size (lbq_attn_d*.hip)
hipError_t launch_attn_d64(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st);
hipError_t launch_attn_d96(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st);
hipError_t launch_attn_d128(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st);
hipError_t launch_attn_d192(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st);
hipError_t launch_attn_d256(const KvAttention &a, const AttnPlan &plan, bool any_short, bool any_long, hipStream_t st);

}  // namespace lbq
