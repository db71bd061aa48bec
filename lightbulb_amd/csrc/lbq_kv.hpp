// lbq_kv.hpp -- the 8-bit paged key/value cache: what its kernels and its C entry points share.
//
// A page holds page_size consecutive tokens of one sequence.  Per (page, kv head) the
// keys lie token by token, [page_size][head_dim] codes, and the values transposed,
// [head_dim][page_size]: each is the order in which the matrix cores take its operand, 8 or
// 16 codes of a lane in one load.  Each (page, kv head) has one scale for its keys and one
// for its values; a value is code * scale.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lbq {

enum : int { KV_INT8 = 0, KV_E4M3 = 1 };
enum : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };  // queries, keys, values and outputs

struct KvCacheView {
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t num_pages;
    int kind, page_size, log2_page, kv_heads, head_dim;
};

struct KvStepView {
    const int32_t *tables;
    int64_t table_stride;
    const int32_t *seq_lens;  // tokens of each sequence, new ones included; 0: none to see
    const int32_t *cu;        // [batch + 1]: sequence b's new tokens are rows cu[b] .. cu[b + 1] - 1
    const int64_t *slots;
    const int32_t *positions;
    int64_t num_tokens;
    int max_blocks, batch;
};

// rows [tokens][heads][head_dim] with any strides (in elements) between tokens and heads
struct KvRows {
    const void *p;
    int64_t token_stride, head_stride;
};

struct KvStepBuild {
    const int32_t *ctx_lens, *new_lens;
    int32_t *tables;
    int64_t table_stride;
    const int32_t *free_pages;
    int64_t num_pages;
    const int32_t *free_count;
    int32_t *free_count_out;
    uint32_t *ticket;  // zero, and left zero; needed where free_count_out == free_count
    int32_t *seq_lens, *cu, *granted;
    int64_t *slots;
    int32_t *positions;
    int64_t num_tokens;
    int batch, max_blocks, log2_page;
};
hipError_t launch_kv_step(const KvStepBuild &a, hipStream_t st);

struct KvRelease {
    int32_t *tables;
    int64_t table_stride;
    const int32_t *lens, *which;
    int32_t *free_pages;
    int64_t num_pages;
    int32_t *free_count;
    int batch, max_blocks, log2_page;
};
hipError_t launch_kv_release(const KvRelease &a, hipStream_t st);

struct KvAppend {
    KvCacheView c;
    KvStepView s;
    int dtype;
    KvRows k, v, q;  // q.p null: no queries to rotate
    void *q_out;     // [num_tokens][q_heads][head_dim]
    int q_heads;
    const float *cos, *sin;  // [max_pos][rot_dim / 2]; rot_dim 0: nothing is rotated
    int64_t max_pos;
    int rot_dim, interleaved;
    int max_new;  // no sequence has more new tokens; 0: not known
};
hipError_t launch_kv_append(const KvAppend &a, hipStream_t st);

struct KvAttention {
    KvCacheView c;
    KvStepView s;             // the keys' side: tables, seq_lens, batch
    const int32_t *cu_q;      // the queries' rows, [batch + 1]
    int64_t num_q;            // rows of q and out
    int dtype, q_heads;
    KvRows q;
    void *out;                // [num_q][q_heads][head_dim]
    float scale;
    int causal;
    int window;               // 0: none
    int max_len;              // no sequence is longer
    int max_new;              // no sequence has more queries; 0: not known
    void *ws;
    size_t ws_bytes;
};
// workgroups of either form that a launch may have (of up to 512 threads: both together below 2^32)
constexpr int64_t MAX_GROUPS = ((int64_t)1 << 22) - 1;
size_t kv_attention_workspace(const KvAttention &a);
hipError_t launch_kv_attention(const KvAttention &a, hipStream_t st);

#ifdef __HIPCC__
// The sequence b of `batch` with start(b) <= x < start(b + 1), for a start that never
// falls and start(0) <= x: 64 probes at a time, so one load's latency per factor of 64 in
// the batch.  The same x in every lane of a wave; all 64 lanes call it.
template <class F>
__device__ __forceinline__ int find_sequence(int batch, int64_t x, F start) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = batch;  // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 63) / 64, i = lo + lane * step;
        const uint64_t below = __ballot(lane * step < n && start(i) <= x) | 1;
        const int at = (63 - __clzll(below)) * step;
        n = min(step, n - at);
        lo += at;
    }
    return lo;
}
#endif

}  // namespace lbq
