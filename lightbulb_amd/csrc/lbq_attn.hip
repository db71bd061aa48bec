// lbq_attn.hip -- attention over the 8-bit paged key/value cache.
#include "lbq_kv.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

namespace lbq {
namespace {

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
__device__ __forceinline__ float code_value(uint8_t c, int kind) {
    return kind == KV_INT8 ? (float)(int8_t)c : __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// o = sum_j softmax_j(scale q . k_j) v_j over the keys j that the query at position pos sees:
// j < len, causal: j <= pos, window w: j > pos - w.  One wave per (query row, head), 64 keys
// at a time with the running maximum and sum: a lane forms one key's product, then holds up
// to four channels of the output.
template <int DT>
__global__ __launch_bounds__(64) void k_attn_simple(KvAttention a) {
    __shared__ float q[256], w[64];
    const int lane = threadIdx.x, D = a.c.head_dim, P = a.c.page_size, H = a.c.kv_heads;
    const int64_t t = blockIdx.x;
    const int hq = blockIdx.y, h = hq / (a.q_heads / H);
    const int b = find_sequence(a.s.batch, t, [&](int i) { return (int64_t)a.cu_q[i]; });
    const int64_t t0 = a.cu_q[b], t1 = a.cu_q[b + 1];
    if (t < t0 || t >= t1) return;  // a row behind the last sequence
    const int64_t len = min((int64_t)a.s.seq_lens[b], (int64_t)a.s.max_blocks * P);
    const int64_t pos = a.s.seq_lens[b] - (t1 - t0) + (t - t0);
    const int64_t hi = a.causal ? min(len, pos + 1) : len;
    const int64_t lo = a.causal && a.window > 0 ? max((int64_t)0, pos - a.window + 1) : 0;
    constexpr int size = DT == DT_F32 ? 4 : 2;
    const char *row = static_cast<const char *>(a.q.p) + (t * a.q.token_stride + hq * a.q.head_stride) * size;
    for (int d = lane; d < D; d += 64) q[d] = load_value<DT>(row, d);
    __syncthreads();
    float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t j0 = lo & ~63ll; j0 < hi; j0 += 64) {
        const int64_t j = j0 + lane;
        const bool seen = j >= lo && j < hi;
        float s = -INFINITY;
        int64_t page = -1;
        if (seen) page = a.s.tables[b * a.s.table_stride + (j >> a.c.log2_page)];
        const bool there = page >= 0 && page < a.c.num_pages;
        if (there) {
            const uint8_t *k = a.c.k + ((page * H + h) * P + (j & (P - 1))) * D;
            float dot = 0.f;
            for (int d = 0; d < D; d++) dot = fmaf(q[d], code_value(k[d], a.c.kind), dot);
            s = dot * a.c.ks[page * H + h] * a.scale;
        }
        float top = s;
#pragma unroll
        for (int d = 32; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
        // (a NaN product stays one: the maximum passes over it, the exponential does not)
        top = fmaxf(m, top);
        const float base = top == -INFINITY ? 0.f : top;
        const float p = there ? expf(s - base) : 0.f, alpha = expf(m - base);
        m = top;
        float ps = p;
#pragma unroll
        for (int d = 32; d; d /= 2) ps += __shfl_xor(ps, d);
        sum = sum * alpha + ps;
        w[lane] = there ? p * a.c.vs[page * H + h] : 0.f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] *= alpha;
        for (int jj = 0; jj < 64; jj++) {
            if (__shfl((int)there, jj) == 0) continue;
            const int64_t pg = __shfl((int)page, jj);
            const uint8_t *v = a.c.v + (pg * H + h) * D * P + ((j0 + jj) & (P - 1));
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (lane + 64 * i < D) o[i] = fmaf(w[jj], code_value(v[(lane + 64 * i) * P], a.c.kind), o[i]);
        }
        __syncthreads();
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < D) store_value<DT>(a.out, (t * a.q_heads + hq) * D + lane + 64 * i, o[i] * inv);
}

}  // namespace

size_t kv_attention_workspace(const KvAttention &) { return 0; }

hipError_t launch_kv_attention(const KvAttention &a, hipStream_t st) {
    const dim3 grid((unsigned)a.num_q, (unsigned)a.q_heads);
    if (a.dtype == DT_F32) k_attn_simple<DT_F32><<<grid, 64, 0, st>>>(a);
    else if (a.dtype == DT_F16) k_attn_simple<DT_F16><<<grid, 64, 0, st>>>(a);
    else k_attn_simple<DT_BF16><<<grid, 64, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace lbq
