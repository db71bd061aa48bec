/*
 * lbq.h -- C ABI of the MI355X quantized-linear library (liblbq.so).
 *
 * This is the drop-in boundary for lightbulb's GGUF quantized-linear path.
 * lightbulb calls QuantizableLinear::Quantized(QMatMul)::forward for every
 * attention/MLP projection and the LM head
 * (/root/reference/src/model/quantizable_linear.rs:36-43, 63-69).  A Rust shim
 * keeps that surface and binds the functions below through `extern "C"`; the
 * binding is plain pointers, 64-bit sizes and an opaque stream pointer, in
 * the style of the reference's only FFI precedent
 * (/root/reference/src/backend/marlin_ffi.rs:84-215), plus status codes.
 *
 * Conventions
 *   - Every function returns 0 (LBQ_OK) or a negative lbq_status, never
 *     aborts; lbq_last_error() gives a thread-local message for the last
 *     failure on the calling thread.
 *   - Pointers named d_* are device pointers (HBM).  `stream` is a
 *     hipStream_t passed as void* (NULL = the null stream); work is ordered
 *     on it and the call does not synchronise unless stated.
 *   - Weights are GGUF blocks in their on-disk byte layout: row-major
 *     [n][k / block_size] blocks, rows contiguous along k
 *     (GGUF ne0 = k; /root/reference/src/gguf/parser.rs:180-199).
 *   - A context owns per-device scratch (quantised activations, the batched
 *     GEMM's workspace, grown on demand, and 64 KiB of its tile counters).  A buffer
 *     that has been outgrown stays until the context goes, for captured graphs that
 *     use it.  Calls that share a context must be
 *     ordered on one stream (the reference runs every forward on one model
 *     thread, src/engine/model_runner.rs:236,383).  Weight handles are
 *     immutable and may be read concurrently.
 */
#ifndef LBQ_H
#define LBQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct lbq_ctx lbq_ctx;
typedef struct lbq_weight lbq_weight;

enum lbq_status {
    LBQ_OK = 0,
    LBQ_ERR_INVALID_ARG = -1,      /* null pointer, negative size, misaligned pointer */
    LBQ_ERR_UNSUPPORTED_TYPE = -2, /* ggml type id not served by this path */
    LBQ_ERR_SHAPE = -3,            /* k not a multiple of the block size, byte count mismatch */
    LBQ_ERR_OOM = -4,              /* device allocation failed */
    LBQ_ERR_HIP = -5,              /* a HIP runtime call failed */
    LBQ_ERR_LIMIT = -6,            /* size beyond a documented maximum */
    LBQ_ERR_FORMAT = -7,           /* malformed or unsupported GGUF container */
    LBQ_ERR_NOT_FOUND = -8,        /* no tensor or metadata key of that name */
    LBQ_ERR_IO = -9                /* a file could not be opened or mapped */
};

/* GGUF/ggml type ids: /root/reference/src/quantization/mod.rs:58-75 (GgmlDType),
 * plus BF16 (30), which candle-core's GgmlDType carries and the reference's own
 * table does not: candle's GGUF reader hands a BF16 tensor to QMatMul::from_qtensor
 * (custom_transformer.rs:358-363), which serves it as its dense variant. */
enum lbq_ggml_type {
    LBQ_TYPE_F32 = 0,  /* dense: an f32 matmul (candle's dense QMatMul variant), k % 8 == 0 */
    LBQ_TYPE_F16 = 1,  /* dense: widened exactly to f32, then as F32 */
    LBQ_TYPE_Q4_0 = 2, /* 32-value blocks, Q8_0 activations */
    LBQ_TYPE_Q4_1 = 3, /* 32-value blocks, Q8_1 activations */
    LBQ_TYPE_Q5_0 = 6, /* 32-value blocks, Q8_0 activations */
    LBQ_TYPE_Q5_1 = 7, /* 32-value blocks, Q8_1 activations */
    LBQ_TYPE_Q8_0 = 8,
    LBQ_TYPE_Q8_1 = 9, /* activation-only type (vec-dot partner of Q4_1/Q5_1) */
    LBQ_TYPE_Q2_K = 10,
    LBQ_TYPE_Q3_K = 11,
    LBQ_TYPE_Q4_K = 12,
    LBQ_TYPE_Q5_K = 13,
    LBQ_TYPE_Q6_K = 14,
    LBQ_TYPE_Q8_K = 15, /* activation-only type (vec-dot partner of the k-quants) */
    LBQ_TYPE_BF16 = 30  /* dense: widened exactly to f32 (bits << 16), then as F32 */
};

/* Thread-local description of the last error on this thread ("" if none). */
const char *lbq_last_error(void);

/* GgmlDType::block_size / type_size (/root/reference/src/quantization/mod.rs:99-126)
 * for the types above (BF16: candle's 1 and 2); 0 for any other id.  lbq_type_size
 * returns the table's value, so GGUF extents computed from it agree with the
 * reference's extract_tensor_bytes (src/quantization/gguf_ops.rs:19-59); for Q2_K
 * that is 82.  (lbq_gguf_tensor_bytes, the mirror of extract_tensor_bytes, still
 * refuses BF16 tensors as the reference's GgmlDType::from_u32 does.) */
int lbq_type_block_size(uint32_t ggml_type);
int lbq_type_size(uint32_t ggml_type);

/* Bytes of one block as it sits in device memory and as the kernels read it
 * (candle's BlockQ2K: scales[16], qs[64], d, dmin): equal to lbq_type_size except
 * for Q2_K, whose block is 84 bytes.  Weight handles take
 * n * (k / block_size) * lbq_type_block_bytes bytes.  No counterpart in the
 * reference, whose table (mod.rs:118) is 2 bytes short for Q2_K. */
int lbq_type_block_bytes(uint32_t ggml_type);

/* Open a context on HIP device `device`.  Replaces the device selection at
 * /root/reference/src/model/parallel_model_manager.rs:239-248. */
int lbq_init(int device, lbq_ctx **out_ctx);
int lbq_ctx_destroy(lbq_ctx *ctx);

/* Upload GGUF blocks (host bytes, on-disk layout, unchanged) to the device
 * and return an immutable weight handle.  Replaces QMatMul::from_qtensor
 * (called at /root/reference/src/model/custom_attention.rs:195-206,
 * mlp_wrapper.rs:127-135, custom_transformer.rs:360-363) together with the
 * upload done by Content::tensor (src/gguf/mod.rs:274-282).
 * nbytes must equal n * (k / block_size) * lbq_type_block_bytes. */
int lbq_weight_create(lbq_ctx *ctx, uint32_t ggml_type, int64_t n, int64_t k, const void *host_blocks,
                      size_t nbytes, lbq_weight **out_w);

/* As lbq_weight_create, but borrows blocks that are already device resident
 * (no copy; the caller keeps the memory alive until lbq_weight_destroy).  Like
 * lbq_weight_create it derives per-row fp16 operand exponents for the batched
 * MFMA GEMM (m > 8) from the block scales, so the blocks must already hold their
 * final contents: the call synchronises the device (whatever writes the blocks,
 * on any stream, completes first) and allocates n bytes for the exponents.  If
 * the caller rewrites the blocks while the handle lives, lbq_weight_refresh must
 * follow before the next forward, or results at m > 8 are wrong (overflowing or
 * underflowing fp16 operands, no error). */
int lbq_weight_wrap_device(lbq_ctx *ctx, uint32_t ggml_type, int64_t n, int64_t k, const void *d_blocks,
                           size_t nbytes, lbq_weight **out_w);

/* Recompute a weight's derived state (the per-row operand exponents above) from
 * its current blocks, stream-ordered on `stream`.  No counterpart in the
 * reference, whose QTensor is immutable; for callers that fill or change the
 * device blocks of a wrapped handle after wrapping it.  A no-op for types and
 * k the MFMA GEMM does not serve (dense weights, k % 256 != 0). */
int lbq_weight_refresh(lbq_weight *w, void *stream);

int lbq_weight_destroy(lbq_weight *w);

/* Shape and type of a weight handle (QTensor::dtype / QTensor::shape). */
int lbq_weight_info(const lbq_weight *w, uint32_t *ggml_type, int64_t *n, int64_t *k);

/* y[m][n] = x[m][k] . W^T in f32 -- QMatMul::forward (candle-core 0.10.2,
 * reached through /root/reference/src/model/quantizable_linear.rs:67).
 * x and y are contiguous f32 device buffers that must not overlap
 * (LBQ_ERR_INVALID_ARG otherwise; the reference returns a new tensor); any
 * leading dims of the reference's [.., k] tensor are flattened into m.  The
 * activation is quantised to Q8_K (k-quant weights), Q8_1 (Q4_1/Q5_1) or Q8_0
 * (the other 32-value types) exactly as the reference CPU path does.
 * Arithmetic by (type, m):
 *   - m <= 8, Q4_K/Q5_K weights of 1024 rows or more up to m = 32 (and
 *     m = 33..64 up to 8192 rows, as two 32-row halves), Q6_K weights with
 *     k > 8192 on the same shapes, Q8_0 weights of 1024 rows or more
 *     (k % 256 == 0) up to m = 32 (m = 33..64 as halves at k <= 8192 up to 8192
 *     rows), and Q4_0/Q4_1/Q5_0/Q5_1 weights of 1024 rows or more (k % 256 == 0)
 *     up to m = 16: each output from integer sub-block dot
 *     products as in the reference (f32 combine; only the summation order
 *     differs, ~1e-7 relative);
 *   - m > 8 otherwise, for every quantised type when k % 256 == 0 (Q4_0, Q4_1,
 *     Q5_0, Q5_1, Q8_0, Q2_K, Q3_K, Q4_K, Q5_K, Q6_K): MFMA on fp16 roundings of
 *     the same activation and weight values (about 4e-4 relative on a row);
 *   - m > 8 with k % 256 != 0: integer block sums on the fp16 matrix cores (the
 *     codes and scales exact in fp16, f32 combine; ~1e-7 relative), with operands
 *     in the context's scratch; where that cannot be had (a graph capture that
 *     would have to grow it, the allocation-free scratch exceeded) the integer
 *     GEMV over chunks of 8 rows.
 * Where the matrix-core decode kernel (m = 2..64) splits a 32-row
 * tile between two workgroups, their halves are added into y with f32 atomic
 * adds when y is plain device memory (hipMalloc; checked once per allocation),
 * else through partial sums in the workspace; either way y = a + b for the two
 * halves, the same bits for finite normal-range halves.  Dense F32/F16/BF16
 * weights are candle's dense variant: no quantisation, an f32 matmul.  At m > 8
 * the 16-bit matrix cores form its products: x as three bf16 operands that add up
 * to it (an F32 weight as three, an F16 weight as two), every product exact (F32: but
 * for one part below 2^-32 of it), sums in f32.  The operands live in memory of the
 * context, a buffer for each stream and for each graph capture, so dense calls
 * need no order with calls on other streams; where there is none (no memory, more
 * than 64 streams, hipStreamPerThread, captures that together would hold 1 GiB), and at
 * k <= 64 with less than 2^22 outputs, the f32 matrix cores run instead.  m == 0 is a no-op. */
int lbq_qmatmul_f32(lbq_ctx *ctx, const lbq_weight *w, const float *d_x, int64_t m, float *d_y, void *stream);

/* lbq_qmatmul_f32's result (the same kernels, the same bits), allocating
 * nothing: no hipMalloc, hipFree or allocating library call.
 * No counterpart in the reference; for callers that cannot allocate device
 * memory -- code under HIP graph capture, tight serving loops, harnesses that
 * forbid it.  The quantised activations and the batched GEMM's workspace live
 * in a fixed array of LBQ_NOALLOC_SCRATCH_BYTES per device (its last 64 KiB
 * are the GEMM's tile counters, zeroed by lbq_init and left zero by every
 * call), resolved by lbq_init and held until the process ends.  A call that needs more (roughly
 * m * k * 2 bytes of fp16 operands plus split-k partials above m = 8; every
 * Llama-3-8B projection fits up to m = 512, down_proj up to m = 2048) returns
 * LBQ_ERR_LIMIT before launching anything; a dense weight's call that needs more
 * runs lbq_qmatmul_f32's form without scratch instead (f32 matrix cores).  All contexts on a device share the
 * one array, which keeps the last call's contents: calls that overlap on one
 * device (on different streams or threads) race and must be ordered by the
 * caller. */
#define LBQ_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)
int lbq_qmatmul_f32_noalloc(lbq_ctx *ctx, const lbq_weight *w, const float *d_x, int64_t m, float *d_y,
                            void *stream);

/* Several weights applied to one x: ys[i][m][n_i] = x . W_i^T, exactly as
 * `count` separate lbq_qmatmul_f32 calls compute them (bit-identical), with x
 * quantised once and, at m = 1, every weight's rows streamed by one launch.
 * Replaces the runs of QMatMul::forward calls on the same input at the q/k/v
 * projections (/root/reference/src/model/custom_attention.rs:265-267) and the
 * gate/up projections (/root/reference/src/model/mlp_wrapper.rs:190,193).
 * 1 <= count <= LBQ_GROUP_MAX; all weights share the ggml type and k. */
#define LBQ_GROUP_MAX 4
int lbq_qmatmul_group_f32(lbq_ctx *ctx, const lbq_weight *const *ws, int count, const float *d_x, int64_t m,
                          float *const *d_ys, void *stream);

/* The gate/up half of the reference's MLP forward (/root/reference/src/model/
 * mlp_wrapper.rs:190-194: `silu(gate_proj.forward(x)) * up_proj.forward(x)`):
 * d_out[m][n] = silu(x . Wg^T) * (x . Wu^T), silu(v) = v / (1 + exp(-v)) in f32.
 * The two products are those of lbq_qmatmul_f32 on the same values.  At
 * m = 1, for Q4_K / Q5_K weights of more than 8192 rows (and more than 32
 * rows per CU) at m = 5..32 -- m = 2..32 when k > 8192 -- (after one activation
 * quantisation), and for the MFMA types but Q4_1 / Q5_1 from m = 256 where tiles of 256
 * rows by 128 outputs keep more than half the CUs busy (after one operand
 * pre-pass), both weights run in one launch and the product is
 * formed in its epilogue, so neither product is written out; otherwise
 * the grouped path fills context memory and one elementwise launch combines it.
 * The m = 2..32 pair launch gives the same bits as that; the one from m = 256 sums each
 * output's k in one piece, and differs in f32 summation order where lbq_qmatmul_f32
 * splits k.  gate and up share the ggml type, n and k. */
int lbq_gate_up_silu_f32(lbq_ctx *ctx, const lbq_weight *w_gate, const lbq_weight *w_up, const float *d_x, int64_t m,
                         float *d_out, void *stream);

/* The RMS norm that precedes those projections (input_layernorm before q/k/v,
 * post_attention_layernorm before gate/up: /root/reference/src/model/
 * custom_transformer_block.rs:329 and the MLP path; candle's RmsNorm in f32:
 * x_norm = x / sqrt(sum(x^2) / k + eps) * norm_w), then the grouped projections or
 * the gate/up product of x_norm.  At m = 1 (k-quants, k <= 8192, x and norm_w
 * 16-byte aligned) the norm and the Q8_K quantisation run in the GEMV prologue
 * -- one launch, x_norm never written.  At m > 1, where every weight reads
 * pre-quantised Q8_K activations (k-quants, k % 256 == 0 up to 16384, x and
 * norm_w 16-byte aligned; m <= 8, or Q4_K/Q5_K weights on the matrix-core batch
 * decode), the norm runs inside the one Q8_K quantisation launch, x_norm again
 * never written.  At m > 8, where every weight runs the MFMA GEMM behind a pre-pass by
 * rows (k % 256 == 0 up to 16384, x and norm_w 16-byte aligned, not the k-sliced kernel
 * of small m), the norm runs inside that pre-pass, with the bits of
 * lbq_rmsnorm_f32 followed by the calls without a norm.  Otherwise x_norm goes to context
 * memory first.  lbq_rmsnorm_f32 is the norm alone. */
int lbq_rmsnorm_f32(const float *d_x, const float *d_w, float eps, int64_t m, int64_t k, float *d_y, void *stream);
int lbq_rmsnorm_qmatmul_group_f32(lbq_ctx *ctx, const lbq_weight *const *ws, int count, const float *d_x,
                                  const float *d_norm_w, float eps, int64_t m, float *const *d_ys, void *stream);
int lbq_rmsnorm_gate_up_silu_f32(lbq_ctx *ctx, const lbq_weight *w_gate, const lbq_weight *w_up, const float *d_x,
                                 const float *d_norm_w, float eps, int64_t m, float *d_out, void *stream);

/* Quantised-activation handle: the two halves of QMatMul::forward as separate
 * calls.  candle's k_quants::matmul first quantises every row of x into
 * vec-dot blocks and then runs vec_dot for all output columns; splitting the
 * two lets call sites that feed one x to several weights -- q/k/v at
 * /root/reference/src/model/custom_attention.rs:265-267, gate/up at
 * mlp_wrapper.rs:190,193 -- quantise x once.  act_type is LBQ_TYPE_Q8_K for
 * k-quant weights, LBQ_TYPE_Q8_0 for Q8_0/Q4_0/Q5_0 weights and LBQ_TYPE_Q8_1
 * for Q4_1/Q5_1 weights.  The handle owns device memory for m rows of k values. */
typedef struct lbq_act lbq_act;
int lbq_act_create(lbq_ctx *ctx, uint32_t act_type, int64_t m, int64_t k, lbq_act **out_act);
int lbq_act_quantize(lbq_act *act, const float *d_x, void *stream);
int lbq_act_destroy(lbq_act *act);
/* y[m][n] from a quantised activation; act's k and vec-dot type must match w. */
int lbq_qmatmul_act_f32(lbq_ctx *ctx, const lbq_weight *w, const lbq_act *act, float *d_y, void *stream);

/* Dequantise the whole weight to f32 [n][k] -- QTensor::dequantize (used at
 * /root/reference/src/model/custom_transformer.rs:323,347 and
 * custom_transformer_block.rs:229,231).  Bit-exact with the reference. */
int lbq_dequantize_f32(lbq_ctx *ctx, const lbq_weight *w, float *d_y, void *stream);

/* Dequantise nelem values of raw device blocks -- dequantize_tensor
 * (/root/reference/src/quantization/mod.rs:158-247), extended to every block type
 * above, and F32 / F16 / BF16 tensors (QTensor::dequantize of the norm weights,
 * custom_transformer_block.rs:229-231, which GGUF files store as F32).
 * nelem must be a multiple of the block size. */
int lbq_dequantize_blocks_f32(uint32_t ggml_type, const void *d_blocks, int64_t nelem, float *d_y, void *stream);

/* Embedding lookup without the dense table: d_out[i][:] = row d_ids[i] of the
 * dequantised weight (f32 [count][k], bit-exact with QTensor::dequantize followed
 * by Embedding::forward's index_select -- custom_transformer.rs:321-323, the
 * token embedding, which the reference dequantises whole at load).  d_ids holds
 * count int32 ids; an id outside [0, n) yields a row of NaN (the reference's
 * index_select raises; the device cannot, so the row is poisoned instead).
 * k must be a multiple of 16; d_out 16-byte aligned. */
int lbq_embedding_f32(lbq_ctx *ctx, const lbq_weight *w, const int32_t *d_ids, int64_t count, float *d_out,
                      void *stream);
/* The same for int64 ids (8-byte aligned), as a tensor library holds them. */
int lbq_embedding_i64_f32(lbq_ctx *ctx, const lbq_weight *w, const int64_t *d_ids, int64_t count, float *d_out,
                          void *stream);

/* Quantise activations x[m][k] to GGUF blocks of `act_type` (LBQ_TYPE_Q8_K:
 * 292-byte blocks; LBQ_TYPE_Q8_0: 34-byte blocks; LBQ_TYPE_Q8_1: 36-byte
 * blocks) -- the activation quantisation inside QMatMul::forward (candle
 * BlockQ8K / BlockQ8_0 / BlockQ8_1 ::from_float).  Exposed so the step can be
 * checked on its own. */
int lbq_quantize_act(uint32_t act_type, const float *d_x, int64_t m, int64_t k, void *d_out_blocks, void *stream);

/* Quantise f32 weights (nelem values, row-major, rows along k) to GGUF blocks
 * of `ggml_type` -- quantize_tensor (/root/reference/src/quantization/mod.rs:257-327),
 * extended to Q5_K/Q6_K and Q4_1/Q5_0/Q5_1.  Runs on the device. */
int lbq_quantize_weights_f32(uint32_t ggml_type, const float *d_w, int64_t nelem, void *d_out_blocks, void *stream);

/* ---------------------------------------------------------------------------
 * 8-bit paged key/value cache and attention over it: what a decoder layer does
 * between its q/k/v projections and its o projection (the reference's
 * custom_attention.rs:250-671 over src/cache/, in f32; here the cache is held in
 * 8 bits).  Four calls make a step:
 *   lbq_kv_step_build    lengths -> block tables, slots and positions, on the device
 *   lbq_kv_append        rotate q and k, quantise k and v into their pages
 *   lbq_kv_attention     prompts, single tokens and cross attention over the pages
 *   lbq_kv_release       pages of finished sequences back to the free ones
 *
 * A page holds page_size (16, 32, 64 or 128) consecutive tokens of one sequence; block j
 * of sequence b, its tokens j * page_size and on, lies in page tables[b][j].  Each
 * (page, kv head) has one scale for its keys and one for its values; a value is
 * code * scale.  Codes are int8 (scale = largest magnitude / 127) or e4m3 (OCP; the
 * power of two that brings the largest magnitude to at most 448); scales are not negative.  A scale grows while its
 * page fills, never falls, and the codes already there are then coded again; a page whose
 * keys or values are not finite has the scale NaN from then on and reads as NaN.
 * head_dim is 64, 96, 128, 192 or 256; dtype is LBQ_TYPE_F32, _F16 or _BF16 and is that of
 * q, k, v and out alike, whose rows [token][head][head_dim] may have any strides (in
 * elements) but the last, which is 1.  All calls run on the context's device; none of them
 * uses the context's memory, so calls on different streams need no order among
 * themselves but that of their own buffers.
 * ------------------------------------------------------------------------- */
enum lbq_kv_kind { LBQ_KV_INT8 = 0, LBQ_KV_E4M3 = 1 };

typedef struct lbq_kv_cache {
    void *d_k;          /* codes [num_pages][kv_heads][page_size][head_dim], 16-byte aligned */
    void *d_v;          /* codes [num_pages][kv_heads][head_dim][page_size], 16-byte aligned */
    float *d_k_scales;  /* [num_pages][kv_heads] */
    float *d_v_scales;  /* [num_pages][kv_heads] */
    int64_t num_pages;
    int32_t kind;       /* lbq_kv_kind */
    int32_t page_size, kv_heads, head_dim;
} lbq_kv_cache;

typedef struct lbq_kv_step {
    const int32_t *d_tables;    /* [batch][table_stride]: pages of each sequence's blocks; an entry that is no page: no keys */
    int64_t table_stride;
    const int32_t *d_seq_lens;  /* [batch]: tokens of each sequence, the new ones included */
    const int32_t *d_cu_new;    /* [batch + 1]: rows cu[b] .. cu[b + 1] - 1 are sequence b's new tokens, its last ones */
    const int64_t *d_slots;     /* [num_tokens]: page * page_size + place of each row, -1: none (append only, else may be NULL) */
    const int32_t *d_positions; /* [num_tokens], -1: none (append only, else may be NULL) */
    int64_t num_tokens;         /* rows of q, k, v and out; those from cu[batch] on are padding and are left as they are */
    int32_t batch;              /* up to 65536 */
    int32_t max_blocks;         /* blocks of a table row in use, <= table_stride */
    int32_t max_len;            /* no seq_lens entry is larger; 0: max_blocks * page_size.  Keys beyond it are not seen */
    int32_t max_new;            /* no sequence has more new tokens; 0: not known.  Rows beyond it are not served */
} lbq_kv_step;

/* Block tables, slots and positions of a step from the requests' lengths, in one launch.
 * Sequence b holds ctx_lens[b] tokens and gets new_lens[b]; its rows are cu_new[b] and on.
 * A sequence is granted its pages if its lengths are not negative, its blocks fit
 * max_blocks and its rows num_tokens, and if it needs none or the pages that it and those
 * before it need are no more than *d_free_count; the i-th page taken is
 * d_free[*d_free_count - 1 - i] and goes into d_tables, whose other entries stay.  Where it is
 * not granted, granted[b] and seq_lens[b] are 0 and its rows' slots and positions -1.
 * A sequence of a negative length counts as one of no rows.
 * *d_free_count_out = *d_free_count less the pages taken; the two pointers may be equal
 * (the step is then taken), in which case d_ticket is a word that is zero before the call and
 * after it.  Where they are not, the pages stay free: their entries in the tables are a forecast, which holds
 * until the next call, and nothing may be appended to their slots.  An entry behind the blocks that a sequence's
 * length needs is of no meaning to any call. */
int lbq_kv_step_build(lbq_ctx *ctx, const int32_t *d_ctx_lens, const int32_t *d_new_lens, int32_t batch,
                      int32_t *d_tables, int64_t table_stride, int32_t max_blocks, int32_t page_size,
                      const int32_t *d_free, int64_t num_pages, const int32_t *d_free_count, int32_t *d_free_count_out,
                      uint32_t *d_ticket, int64_t num_tokens, int32_t *d_seq_lens, int32_t *d_cu_new, int32_t *d_granted,
                      int64_t *d_slots, int32_t *d_positions, void *stream);

/* The pages that hold the lens[b] tokens of each sequence with which[b] != 0 go back on top of
 * the free ones, sequence by sequence and block by block, and their table entries become -1
 * (so a second release of the same sequence frees nothing).  A page that stands in two released
 * tables goes back twice: sequences that share pages are released with all but one of the shared
 * entries at -1. */
int lbq_kv_release(lbq_ctx *ctx, const int32_t *d_lens, const int32_t *d_which, int32_t batch, int32_t *d_tables,
                   int64_t table_stride, int32_t max_blocks, int32_t page_size, int32_t *d_free, int64_t num_pages,
                   int32_t *d_free_count, void *stream);

/* k and v [num_tokens][kv_heads][head_dim] into their pages, after the rotation of k's first
 * rot_dim channels by its row's position where rot_dim > 0; and, where d_q is not NULL, q's
 * rows rotated likewise into d_q_out [num_tokens][q_heads][head_dim] (contiguous, apart from
 * q, k and v).  Pairs are the channels (i, i + rot_dim / 2), or neighbours where interleaved;
 * (a, b) becomes (a cos - b sin, b cos + a sin), with cos and sin [max_pos][rot_dim / 2] f32.
 * A position from max_pos on gives NaN.  Each page takes new tokens of one sequence only; the first of
 * a sequence's new rows in a page gives the page (its slot), and where that is -1 or not the place
 * that seq_lens and cu_new say, none of them is written.  Rows of q whose position is -1 are passed
 * over. */
int lbq_kv_append(lbq_ctx *ctx, const lbq_kv_cache *cache, const lbq_kv_step *step, uint32_t dtype, const void *d_k,
                  int64_t k_token_stride, int64_t k_head_stride, const void *d_v, int64_t v_token_stride,
                  int64_t v_head_stride, const void *d_q, int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads,
                  const float *d_cos, const float *d_sin, int64_t max_pos, int32_t rot_dim, int32_t interleaved,
                  void *d_q_out, void *stream);

/* out[t][h] = sum_j softmax_j(scale * q[t][h] . k[j]) v[j] over the cached tokens j of row t's
 * sequence, kv head h / (q_heads / kv_heads).  causal: row i of n new ones is at position
 * seq_len - n + i and sees j <= position, and with a window > 0 only j > position - window.
 * Not causal (window 0): every row sees the whole sequence -- cross attention, with cu_new of
 * the decoder's rows and tables and seq_lens of the encoder's states.  A row that sees
 * nothing is zero; one that sees something and whose query is not finite is NaN.  out is [num_tokens][q_heads][head_dim], contiguous, apart from q.
 * Sums and softmax are f32.  Queries go into their products off by 2^-22 of themselves or 2^-31 of their row's
 * largest.  Weights go into their product with the values relative to the row's
 * largest weight with its value scale, as f16 in two parts (f32, f16: off by 2^-22 of themselves or 2^-34 of the
 * largest) or one (bf16: 2^-11); value scales below 2^-80 of the sequence's largest count as that.  f32
 * results are f32's, about 1e-6 of sum_j softmax_j |v_j|.  The work of one sequence is spread over the chip through d_ws:
 * lbq_kv_attention_workspace gives the bytes that are of use; with less (or NULL) the same
 * call runs with less of it spread. */
int lbq_kv_attention_workspace(lbq_ctx *ctx, const lbq_kv_cache *cache, const lbq_kv_step *step, int32_t q_heads,
                               size_t *bytes);
int lbq_kv_attention(lbq_ctx *ctx, const lbq_kv_cache *cache, const lbq_kv_step *step, uint32_t dtype, const void *d_q,
                     int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads, float scale, int32_t causal,
                     int64_t window, void *d_out, void *d_ws, size_t ws_bytes, void *stream);

/* ---------------------------------------------------------------------------
 * Linears in 8-bit integers with a scale for each token and channel, and the norms between
 * them.  A token's values x[k] become int8 codes and one f32 scale:
 *   scale = max_j |x[j]| / 127 rounded to f32, at least 2^-126; 0 where all values are 0
 *   code  = x / scale to the nearest whole number, ties to even, as if the quotient were exact
 * A token with a value that is not finite has the scale NaN and codes 0: its products are NaN.
 * A weight has int8 codes [n][k] and one f32 scale for each of its n channels.  An output is
 *   y[i][j] = scale[i] * channel_scale[j] * sum_k code[i][k] weight_code[j][k] + bias[j]
 * with the sum exact (k is at most 131071, codes may be -128); the sum and the scales' product are rounded to
 * f32, and their product with the bias added is rounded once.  Where a scale is outside 2^-60 to 2^44, 0 too,
 * all is formed in 64 bits.  The same bits come out whatever m is and wherever the row stands.
 * Rows of codes, of tokens and weights alike, are LBQ_I8_ROW(k) bytes apart and zero from k on, 16-byte
 * aligned.  Types are LBQ_TYPE_F32, _F16 or _BF16; rows of values may have any stride (in elements).  Up to
 * 2^22 - 1 tokens and 2^24 channels a weight, tokens times channels of a call below 2^35.  Results lie apart from
 * the inputs (weights, biases and norms' vectors among them) and from each other; others are refused.
 * All calls run on the context's device and use none of its memory: calls on different streams need
 * no order among themselves but that of their own buffers.
 * ------------------------------------------------------------------------- */
#define LBQ_I8_ROW(k) (((int64_t)(k) + 127) / 128 * 128)

typedef struct lbq_i8_weight {
    const int8_t *d_codes;  /* [n][LBQ_I8_ROW(k)] */
    const float *d_scales;  /* [n] */
    const float *d_bias;    /* [n], or NULL */
    int64_t n;
} lbq_i8_weight;

/* x[m][k] -> codes [m][LBQ_I8_ROW(k)] and scales [m].  Weights' rows are quantised by the same call. */
int lbq_i8_quantize(lbq_ctx *ctx, uint32_t type, const void *d_x, int64_t row_stride, int64_t m, int64_t k,
                    int8_t *d_codes, float *d_scales, void *stream);

/* d_ys[i][m][n_i] of `count` weights (up to LBQ_GROUP_MAX) on one set of tokens: q, k and v, say.  d_x NULL:
 * d_codes and d_scales hold the tokens.  Else x[m][k] of x_type is quantised first, into d_codes and
 * d_scales, whose contents then are not the caller's; up to LBQ_I8_FUSED_ROWS tokens of together at most
 * LBQ_I8_FUSED_CODES bytes of codes (m rounded up to a power of two) are quantised by the product's kernel where
 * the weights have at most LBQ_I8_FUSED_CHANNELS channels in all, and d_codes and d_scales may be NULL. */
#define LBQ_I8_FUSED_ROWS 4
#define LBQ_I8_FUSED_CODES 16384
#define LBQ_I8_FUSED_CHANNELS 16384
int lbq_i8_linear(lbq_ctx *ctx, uint32_t x_type, const void *d_x, int64_t x_stride, int8_t *d_codes, float *d_scales,
                  int64_t m, int64_t k, const lbq_i8_weight *const *ws, int count, uint32_t out_type, void *const *d_ys,
                  void *stream);

/* d_y[m][n] = silu(g) * u of the two weights' products g and u (f32, biases included), silu(v) =
 * v / (1 + exp(-v)), as an f32 value down to its least one: mlp_wrapper.rs:190-194 over such weights, which have
 * the same n and k. */
int lbq_i8_gate_up_silu(lbq_ctx *ctx, uint32_t x_type, const void *d_x, int64_t x_stride, int8_t *d_codes,
                        float *d_scales, int64_t m, int64_t k, const lbq_i8_weight *gate, const lbq_i8_weight *up,
                        uint32_t out_type, void *d_y, void *stream);

/* The residual stream's update by a block's output x[m][k] and the norm in front of the next block:
 *   r = residual + scale * gate * post(x)        y = norm(r)
 * residual, gate and the norms may each be NULL (nothing is added; no gate; no norm).  A norm is
 *   LBQ_NORM_RMS    u / sqrt(mean(u^2) + eps) * (weight + offset) + bias
 *   LBQ_NORM_LAYER  the same of u - mean(u)
 * with f32 weight and bias (may be NULL) of k values.  The gate is of x's type, gate_stride elements from row to
 * row, 0: one for all.  r [m][k] is of residual_type and y [m][k] of x's, both contiguous; with d_codes and
 * d_scales y becomes codes, of its values rounded to f32, and d_y is NULL.  d_r may be NULL, or d_residual
 * itself where its rows are contiguous.  Sums over a row are in 64 bits, values in 32, or 64 where y becomes
 * codes; y is the norm of r before r is rounded to its type.  k is at most 32768. */
enum lbq_norm_kind { LBQ_NORM_RMS = 0, LBQ_NORM_LAYER = 1 };
typedef struct lbq_norm {
    int32_t kind; /* lbq_norm_kind */
    float eps, offset;
    const float *d_weight, *d_bias;
} lbq_norm;
int lbq_residual_norm(lbq_ctx *ctx, uint32_t type, const void *d_x, int64_t x_stride, uint32_t residual_type,
                      const void *d_residual, int64_t residual_stride, const lbq_norm *post, const void *d_gate,
                      int64_t gate_stride, float scale, const lbq_norm *norm, int64_t m, int64_t k, void *d_r, void *d_y,
                      int8_t *d_codes, float *d_scales, void *stream);

/* ---------------------------------------------------------------------------
 * GGUF container (v3, little-endian) and the direct GGUF -> device upload.
 * lbq_gguf_open maps the file and parses it as the reference's parse_gguf does
 * (/root/reference/src/gguf/parser.rs:136-213, reached from Content::read,
 * src/gguf/mod.rs:62-92): magic, version 3 only, metadata (types 0..12, arrays),
 * tensor infos, data section at the infos' end rounded up to general.alignment
 * (UInt32; default 32).  Every read is bounds-checked: a malformed file gives
 * LBQ_ERR_FORMAT with the reference's message, never a fault.  Parsing and the
 * byte accessors are host-only.  Strings returned point into the handle and live
 * until lbq_gguf_close.
 * ------------------------------------------------------------------------- */
typedef struct lbq_gguf lbq_gguf;
int lbq_gguf_open(const char *path, lbq_gguf **out);
int lbq_gguf_close(lbq_gguf *g);
/* GGUFHeader fields (parser.rs:112-121) and the file size; any pointer may be NULL. */
int lbq_gguf_header(const lbq_gguf *g, uint32_t *version, int64_t *tensor_count, int64_t *metadata_count,
                    uint64_t *alignment, uint64_t *tensor_data_offset, uint64_t *file_size);
/* TensorInfo of tensor `index` in file order (parser.rs:103-109): name, ggml type,
 * dims (ne0 first; dims must hold n_dims <= 8 values), offset within the data section. */
int lbq_gguf_tensor_info(const lbq_gguf *g, int64_t index, const char **name, uint32_t *ggml_type, uint32_t *n_dims,
                         uint64_t *dims, uint64_t *offset);
int lbq_gguf_find_tensor(const lbq_gguf *g, const char *name, int64_t *index);
/* A tensor's bytes in the mapped file, as extract_tensor_bytes
 * (src/quantization/gguf_ops.rs:19-59): ceil(numel / block_size) * type_size
 * bytes at data_offset + offset, for every GgmlDType (quantization/mod.rs:58-127). */
int lbq_gguf_tensor_bytes(const lbq_gguf *g, const char *name, const void **data, size_t *nbytes);
/* Metadata (parser.rs:24-81): key and MetadataValueType by index; typed reads by
 * key (integers of any width and bool; f32/f64; strings; array element type and
 * length).  A missing key gives LBQ_ERR_NOT_FOUND, a type mismatch LBQ_ERR_FORMAT. */
int lbq_gguf_meta_key(const lbq_gguf *g, int64_t index, const char **key, uint32_t *value_type);
int lbq_gguf_meta_int(const lbq_gguf *g, const char *key, int64_t *out);
int lbq_gguf_meta_float(const lbq_gguf *g, const char *key, double *out);
int lbq_gguf_meta_string(const lbq_gguf *g, const char *key, const char **data, size_t *len);
int lbq_gguf_meta_array(const lbq_gguf *g, const char *key, uint32_t *elem_type, uint64_t *len);
/* Copy a tensor's blocks into device memory through pinned staging (synchronous):
 * ceil(numel / block_size) * lbq_type_block_bytes bytes -- the extent above except
 * for Q2_K, whose GgmlDType entry (82 bytes) is shorter than its 84-byte block. */
int lbq_gguf_copy_tensor(const lbq_gguf *g, const char *name, void *d_dst, size_t dst_bytes);
/* A weight handle straight from the file: the tensor (2-D, ne0 = k, ne1 = n, a
 * served type) goes through pinned staging into device memory the handle owns.
 * Replaces Content::tensor -> QMatMul::from_qtensor (src/gguf/mod.rs:274-282 and
 * the call sites listed at lbq_weight_create). */
int lbq_weight_from_gguf(lbq_ctx *ctx, const lbq_gguf *g, const char *name, lbq_weight **out_w);

#ifdef __cplusplus
}
#endif
#endif /* LBQ_H */
