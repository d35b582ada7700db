/*
 * qlinear_b200.h -- C ABI of libqlinear_b200.so, the B200 (sm_100a) block-quantized
 * linear path of the local-llm engine (allenzhang61/blog, AI/codes/local-llm).
 *
 * Every entry point below is the C twin of one reference launch function in
 * src/backend/cuda/ops/kernel.cuh (cited per function): same argument order and
 * meaning, raw GGUF weight bytes as uploaded unchanged by CudaWeightPool
 * (CudaWeightPool.cpp:148-175), fp32 activations, launches on the library's
 * current stream (the reference's process-global stream, common.cpp:12-17).
 * Differences from the reference, by design:
 *   - each function returns a status instead of void; an unsupported dtype or
 *     an invalid shape returns QL_EINVAL instead of silently doing nothing
 *     (the reference's launchers fall through `default: break;`, launch.cu:57-58);
 *   - Q4_0 is supported (the reference parses it but has no arithmetic for it);
 *   - all pointers are device pointers unless stated otherwise.
 * A C++ header-only shim with the reference's exact C++ signatures
 * (DType enum, void return, throw on error) is in qlinear_b200_launch.hpp.
 */
#ifndef QLINEAR_B200_H
#define QLINEAR_B200_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define QL_API __attribute__((visibility("default")))
#else
#define QL_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* GGML type codes, equal to the reference's DType (src/tensor/TensorCommon.h:15-33). */
#define QL_F32 0
#define QL_F16 1
#define QL_Q4_0 2
#define QL_Q5_0 6
#define QL_Q8_0 8
#define QL_Q4_K 12
#define QL_Q6_K 14
#define QL_BF16 30 /* activations of the ql_kv8_* calls only */

/* Status codes. */
#define QL_OK 0
#define QL_EINVAL 1   /* bad argument: dtype, shape, block multiple, null pointer */
#define QL_ECUDA 2    /* CUDA runtime error (see ql_last_error) */
#define QL_EDEVICE 3  /* a kernel gave up a bounded wait and recorded an error */

/* ---- runtime -------------------------------------------------------------------- */
/* set/get the stream every launch uses (reference set/get_current_cuda_stream,
 * common.h:40-44).  NULL = the legacy default stream. */
QL_API int ql_set_stream(void *stream);
QL_API void *ql_get_stream(void);
/* Allocate the per-device workspace (stream-K partials, arrival counters, argmax
 * partials, error word) for `device`.  Called implicitly by the first launch on a
 * device; call it explicitly before capturing launches into a CUDA graph. */
QL_API int ql_init(int device);
/* Human-readable description of the last error returned by this thread. */
QL_API const char *ql_last_error(void);
/* Synchronize the current stream and read (and clear) the device error word. */
QL_API int ql_check_device(void);

/* ---- quantized linear (reference kernel.cuh:34-43) ------------------------------- */
/* y[m, o] = sum_k W[o, k] * x[m, k].  W: out_dim rows of row_bytes GGUF bytes.
 * x: [m, in_dim] f32, y: [m, out_dim] f32, row-major.  kernel.cuh:34-35. */
QL_API int ql_quant_gemv(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const float *x, float *y,
                  int out_dim, int in_dim, int m);
/* y[o] += W[o, :] . x  (m = 1).  kernel.cuh:37-38. */
QL_API int ql_quant_gemv_add(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const float *x, float *y,
                      int out_dim, int in_dim);
/* Same contract as ql_quant_gemv, intended for m > 1 (prefill).  kernel.cuh:42-43. */
QL_API int ql_quant_matmul(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const float *x, float *y,
                    int out_dim, int in_dim, int m);
/* Prefill GEMM with a selectable path and fused extras (no reference twin; the
 * reference runs prefill as launch_quant_matmul, kernel.cuh:42-43, or as
 * dequantize-to-f16 + cuBLAS, TensorTool.cpp:127-144):
 *   y[m, o] (+)= scale_m * sum_k W[o, k] * g[k] * x[m, k] + bias[o]
 * with x rows x_stride floats apart, y rows y_stride apart, optional fused RMSNorm
 * (gamma != NULL: scale_m = 1/sqrt(mean_k x[m,k]^2 + eps), g = gamma; else 1),
 * optional bias, accumulate != 0 adds into y.  path: QL_PATH_AUTO picks by shape;
 * QL_PATH_GEMV forces the CUDA-core streaming engine (fp32 activations, exact
 * decode); QL_PATH_TENSOR forces the tcgen05 tensor-core GEMM (Q4_K, Q4_0 or Q8_0, in_dim
 * a multiple of 256; activations and dequantized weights rounded to f16, fp32
 * accumulation; QL_EINVAL when the shape or dtype does not qualify). */
#define QL_PATH_AUTO 0
#define QL_PATH_GEMV 1
#define QL_PATH_TENSOR 2
QL_API int ql_quant_matmul_ex(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const float *x,
                              int64_t x_stride, float *y, int64_t y_stride, int out_dim, int in_dim, int m,
                              const float *gamma, float eps, const float *bias, int accumulate, int path);
/* Greedy LM head (fused GEMV/GEMM + argmax, no separate argmax launch): for each token m,
 * out_idx[m] = index_offset + argmax_o y[m, o] with y as ql_quant_matmul_ex (plain store,
 * optional fused RMSNorm), lowest index on ties, NaN never wins (reference argmax,
 * kernel.cu:3531-3592).  logits (nullable) also receives y.  out_key (nullable) receives
 * an order-preserving 64-bit key per token (larger = better, ties to the lower index);
 * the maximum key over vocabulary shards, each launched with its own index_offset,
 * selects the same token as an argmax over the whole vocabulary.  m <= 4096. */
QL_API int ql_quant_gemv_argmax_ex(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const float *x,
                                   int64_t x_stride, float *logits, int64_t logits_stride, int out_dim, int in_dim,
                                   int m, const float *gamma, float eps, int index_offset, int *out_idx,
                                   uint64_t *out_key);
/* ---- a chain of single-token GEMVs in one persistent launch ----------------------
 * A decode step's projections (q/k/v, o + residual, gate/up SwiGLU, down + residual,
 * ..., LM head + argmax) as one cooperative kernel: the weight stream runs across op
 * boundaries and each op waits at a grid barrier for the previous op's output.  Q4_K,
 * one token, in_dim a multiple of 256 and >= 1792, 16-byte aligned weights with
 * row_bytes % 16 == 0 and >= 32 rows per source.  Op semantics equal the per-op entry
 * points: STORE y = (RMSNorm?)(x) . W^T + bias over 1..3 stacked sources (all but the
 * last a multiple of 32 rows), optionally with a greedy argmax (argmax_idx, device int,
 * index + argmax_offset; y may then be NULL); ADD y += ...; SWIGLU y = SiLU(g) * u with
 * w[0] = gate, w[1] = up.  Every op may read what any earlier op wrote.  The chain keeps
 * the pointers: buffers must outlive it.  ql_gemv_chain_run enqueues one launch on the
 * current stream (graph-capturable). */
#define QL_OP_STORE 0
#define QL_OP_ADD 1
#define QL_OP_SWIGLU 2
/* MLP (one GPU): y += down . (SiLU(gate . x^) * (up . x^)), x^ = RMSNorm(x) with gamma, as SWIGLU
 * then ADD in one op without the grid barrier between them: w[0] = gate, w[1] = up (rows[0] =
 * rows[1] = FFN width, a multiple of 256), w[2] = down (rows[2] = len(y), in FFN blocks).  The
 * down projection is split over the FFN (two SMs per 256-row chunk) and its partial sums are
 * added in 64-bit fixed point (2^-32 resolution, |y| < 2^31; deterministic).  y must be last
 * written by an ADD op of the chain (same y and rows), and the next op must not be an ADD into
 * y or another MLP.  The SwiGLU activations are not stored. */
#define QL_OP_MLP 3
typedef struct ql_chain_op {
    int32_t kind;
    int32_t quant_type;
    int32_t nsrc;
    const uint8_t *w[3];
    size_t row_bytes[3];
    int32_t rows[3];
    int32_t in_dim;
    const float *x;
    const float *gamma;
    float eps;
    const float *bias;
    float *y;
    int *argmax_idx;
    int32_t argmax_offset;
    int32_t reduce; /* tensor parallel ADD: y += sum over ranks of this op's partial (no bias) */
    /* batched chains only (ql_gemv_chain_create_batch): floats between consecutive tokens' rows of
     * x and of y; 0 = rows packed (in_dim, resp. the op's total output rows) */
    int64_t x_stride;
    int64_t y_stride;
    /* RoPE fused into a STORE op (no reference twin as a fusion; the reference rotates q and k in
     * its attention kernels, kernel.cu:186-260): output rows [0, rope_rows) -- whole heads of
     * head_dim rows, e.g. the q and k rows of a stacked q/k/v -- are rotated after bias, pairing
     * rows i and i + head_dim/2 of each head: (x1, x2) -> (x1 c - x2 s, x2 c + x1 s), angle =
     * pos / rope_theta^(2i / head_dim).  rope_pos: device int32, the position (batched chains: one
     * per token).  rope_rows = 0 disables it; head_dim a multiple of 32, at most 128 in batched
     * chains; no argmax on a RoPE op. */
    const int32_t *rope_pos;
    float rope_theta;
    int32_t rope_rows;
    int32_t head_dim;
} ql_chain_op;
QL_API int ql_gemv_chain_create(const ql_chain_op *ops, int nops, void **chain);
/* Tensor-parallel chain: ops with reduce != 0 (row-parallel ADD projections) sum their
 * partials over ranks inside the kernel through peer memory (each rank's exchange buffer,
 * ql_gemv_chain_exchange_bytes bytes, zeroed, mapped into every rank: exchange[r] for
 * rank r, e.g. with ql_ipc_alloc / ql_ipc_open); an argmax op (vocabulary shard with
 * argmax_offset) combines the ranks' keys the same way.  Every rank must create and run
 * the same chain; a rank that never arrives makes the others give up after ~5 s with an
 * error in the device error word. */
QL_API size_t ql_gemv_chain_exchange_bytes(const ql_chain_op *ops, int nops, int world);
QL_API int ql_gemv_chain_create_tp(const ql_chain_op *ops, int nops, int rank, int world, void *const *exchange,
                                   void **chain);
/* Device allocation shareable with other processes (zeroed), its CUDA IPC handle, and the
 * peer side: map / unmap another process's allocation. */
QL_API int ql_ipc_alloc(size_t bytes, void **ptr, uint8_t *handle);
QL_API int ql_ipc_free(void *ptr);
QL_API int ql_ipc_open(const uint8_t *handle, void **ptr);
QL_API int ql_ipc_close(void *ptr);
/* Batched chain (no reference twin; the reference runs batched decode as quant_matmul_kernel,
 * kernel.cu:1253-1279, one warp per (token, row) on the CUDA cores): the same op list for
 * `tokens` (1..32) tokens in one persistent launch on the tensor cores.  x and y are [tokens, *]
 * row-major with the ops' x_stride / y_stride; RMSNorm, bias, residual add and SwiGLU apply per
 * token; an argmax op writes one index per token (argmax_idx[0..tokens)).  Kinds STORE, ADD,
 * SWIGLU (no MLP, no tensor-parallel reduce); Q4_K; stacked sources but the last a multiple of
 * 128 rows; x rows 16-byte aligned.  Weights and x * gamma are rounded to f16 (|x * gamma| <
 * 65504), accumulation is fp32.  ql_gemv_chain_run / ql_gemv_chain_destroy run and free it. */
QL_API int ql_gemv_chain_create_batch(const ql_chain_op *ops, int nops, int tokens, void **chain);
QL_API int ql_gemv_chain_run(void *chain);
QL_API int ql_gemv_chain_destroy(void *chain);

/* Reserve the tensor-core path's scratch (f16 activations, row scales, split-K
 * partial tiles) on the current device for up to max_tokens x max_in_dim, so later
 * prefill calls of at most that size allocate nothing (e.g. inside graph capture).
 * Larger calls grow the scratch with cudaMalloc. */
QL_API int ql_reserve_prefill(int max_tokens, int max_in_dim);

/* ---- tensor-parallel exchange over NVLink peer memory ------------------------------
 * One-shot all-reduce for the decode step's row-parallel projections (no reference
 * twin: the reference engine is single-GPU).  Setup, once per rank:
 *   ql_comm_alloc   allocates this rank's zeroed exchange buffer on the current device
 *                   and returns its CUDA IPC handle (QL_IPC_HANDLE_BYTES bytes);
 *   (exchange the handles between ranks by any host channel, in rank order)
 *   ql_comm_create  maps every peer's buffer (handles: world x QL_IPC_HANDLE_BYTES).
 * Per step: the same sequence of ql_allreduce_f32 calls on every rank, each naming
 * its call site with a distinct slot < slots, then one ql_comm_step.  Everything is
 * enqueued on the current stream and may be captured into a CUDA graph.  A peer that
 * never arrives makes the call give up after ~5 s with an error in the device error
 * word (ql_check_device returns QL_EDEVICE). */
#define QL_IPC_HANDLE_BYTES 64
QL_API size_t ql_comm_bytes(int world, int max_floats, int slots);
QL_API int ql_comm_alloc(int world, int max_floats, int slots, void **exchange, uint8_t *handle);
QL_API int ql_comm_create(int rank, int world, int max_floats, int slots, void *exchange, const uint8_t *handles,
                          void **comm);
QL_API int ql_comm_destroy(void *comm);
/* buf[0..n) (device, n <= max_floats) := sum over ranks, bit-identical on every rank. */
QL_API int ql_allreduce_f32(void *comm, float *buf, int n, int slot);
QL_API int ql_comm_step(void *comm);

/* act[f] = SiLU(Wg[f] . x) * (Wu[f] . x).  kernel.cuh:65-67. */
QL_API int ql_quant_swiglu(int32_t quant_type, const uint8_t *gate_weight, const uint8_t *up_weight,
                    size_t gate_row_bytes, size_t up_row_bytes, const float *x, float *act, int ffn_dim,
                    int in_dim);

/* ---- MoE (reference kernel.cuh:72-76, 125-129, 335-336) -------------------------- */
/* act[r, f] = SiLU(Wg[e_r][f] . x) * (Wu[e_r][f] . x), e_r = expert_ids[r] (device);
 * e_r < 0 writes zeros.  Expert e's rows start at weight + e * expert_bytes. */
QL_API int ql_quant_swiglu_indexed(int32_t quant_type, const uint8_t *gate_weight, const uint8_t *up_weight,
                            size_t gate_expert_bytes, size_t up_expert_bytes, size_t gate_row_bytes,
                            size_t up_row_bytes, const float *x, const int *expert_ids, float *act, int k,
                            int ffn_dim, int in_dim);
/* out[h] += sum_r route_weights[r] * (Wd[e_r][h] . act[r, :]) over routes with e_r >= 0,
 * in a fixed (deterministic) order. */
QL_API int ql_quant_down_f32_indexed_accum_ordered(int32_t quant_type, const uint8_t *down_weight,
                                            size_t down_expert_bytes, size_t down_row_bytes, const float *act,
                                            const int *expert_ids, const float *route_weights, float *out, int k,
                                            int hidden_size, int ffn_dim);
/* Per token: softmax over n_experts (<= 64) logits, top-k by logit (lowest id on
 * ties, non-finite = -inf), top_w = p * routed_scaling. */
QL_API int ql_moe_router_topk(const float *router_logits, int *top_idx, float *top_w, int tokens, int n_experts, int k,
                       float routed_scaling);

/* Grouped routed experts for a batch of tokens (no reference twin: the reference runs
 * ql_quant_swiglu_indexed and ql_quant_down_f32_indexed_accum_ordered once per token,
 * RoutedExperts.cpp:80-118).  Every expert's rows are read once per call for all the tokens
 * routed to it.  Route (t, r) has expert id expert_ids[t * k + r]; it belongs to this call when
 * e = id - expert_begin is in [0, n_experts) (expert e's rows start expert_bytes * e past the
 * weight pointer: one expert-parallel shard of experts), and is skipped otherwise.
 *   act[t * k + r][f] = SiLU(Wg[e][f] . x_t) * (Wu[e][f] . x_t), 0 for a skipped route,
 * x_t = x + t * x_stride, act rows ffn_dim floats apart.  Numerics as QL_PATH_TENSOR: each
 * activation row (times a power of two) and each dequantized weight rounded to f16, fp32
 * accumulation on the tensor cores.  Q4_0, Q5_0, Q8_0, Q4_K; rows up to ~3.5 KB and up to 256
 * experts per call run grouped (16 rows per warp in shared memory), others run the per-token
 * indexed launches. */
QL_API int ql_moe_swiglu_grouped(int32_t quant_type, const uint8_t *gate_weight, const uint8_t *up_weight,
                                 size_t gate_expert_bytes, size_t up_expert_bytes, size_t gate_row_bytes,
                                 size_t up_row_bytes, const float *x, int64_t x_stride, const int *expert_ids,
                                 int expert_begin, int n_experts, float *act, int tokens, int k, int ffn_dim,
                                 int in_dim);
/* out[t][h] += total_t,h with total = fmaf(Wd[e][h] . act[t * k + r], route_weights[t * k + r],
 * total) over t's routes r = 0..k-1 that belong to this call, in route order (the reference
 * combine, kernel.cu:2252-2287); out rows out_stride floats apart.  Same numerics and limits
 * as ql_moe_swiglu_grouped. */
QL_API int ql_moe_down_grouped_accum_ordered(int32_t quant_type, const uint8_t *down_weight, size_t down_expert_bytes,
                                             size_t down_row_bytes, const float *act, const int *expert_ids,
                                             int expert_begin, int n_experts, const float *route_weights,
                                             float *out, int64_t out_stride, int tokens, int k, int hidden,
                                             int ffn_dim);

/* ---- decode attention around the projections (reference kernel.cuh:185-194) ------- */
/* Causal attention with an output gate for the token at position *pos_dev (device int, so a
 * captured launch replays at every step): for query head h (kv head h / (n_heads / kv_heads)),
 *   attn_h = softmax_j((q_h . k_j) / sqrt(head_dim)) . v_j * sigmoid(gate_h),  j = 0..pos,
 * q, gate, attn [n_heads * head_dim]; key_cache / value_cache [max_seq_len][kv_heads][head_dim],
 * bf16 when kv_bf16 != 0, else f32 (launch_full_attention_attend, launch.cu:676-692).  Keys are
 * split over CTAs per KV head (each K/V tile read once for the head's whole query group) and the
 * splits merged by a second launch.  head_dim <= 256. */
QL_API int ql_full_attention_attend(const float *q, const float *gate, const void *key_cache,
                                    const void *value_cache, int kv_bf16, float *attn, int n_heads, int kv_heads,
                                    int head_dim, int max_seq_len, const int *pos_dev);
/* The same for `tokens` queries at positions start_pos .. start_pos + tokens - 1, rows
 * n_heads * head_dim apart (launch_full_attention_attend_batch, launch.cu:694-709). */
QL_API int ql_full_attention_attend_batch(const float *q, const float *gate, const void *key_cache,
                                          const void *value_cache, int kv_bf16, float *attn, int tokens, int n_heads,
                                          int kv_heads, int head_dim, int max_seq_len, int start_pos);

/* ---- 8-bit KV cache (no reference twin; the reference's cache is f32 or bf16, read by
 *      ql_full_attention_attend) --------------------------------------------------------
 * What a serving step does between the q/k/v projection and the attention's output, over a paged
 * cache of one byte per value.  A page holds QL_KV8_BLOCK tokens of every KV head; a full page has one
 * f32 scale per KV head for K and one for V:
 *   scale = max|x| / 127 over the page's tokens and the head's dimensions (>= 0), byte = rint(x / scale) + 128
 * (x / scale kept within +-127, which a subnormal scale may pass; scale 0: bytes 128; a page that holds NaN or
 * infinity has a NaN scale).  The tokens of a sequence's last, unfinished page are exact: their rows stand in f32 in
 * the "open" rows, from which the page is quantised once, when it is full.  So the bytes do not depend on how a
 * sequence was cut into calls.  kv_len may go back between calls (rejected speculative tokens): to any length within
 * the last two pages of the longest the sequence has been, whose rows the open rows hold (at least QL_KV8_BLOCK tokens
 * less than the longest), and to any multiple of QL_KV8_BLOCK.
 * All buffers are the caller's device memory; every base is 16-byte aligned.  head_dim: a multiple of 32
 * up to 256; activations f32 (QL_F32) or bf16 (QL_BF16).  kv_len, q_start, page_table and slots are read
 * on the device, so a captured CUDA graph follows them.  A page, slot, length or position outside the
 * given extents is not accessed, and is reported by the next ql_check_device (QL_EDEVICE). */
#define QL_KV8_BLOCK 32
typedef struct ql_kv8_cache {
    uint8_t *k_codes, *v_codes;  /* [n_pages][kv_heads][QL_KV8_BLOCK][head_dim] */
    float *k_scale, *v_scale;    /* [n_pages][kv_heads] */
    float *k_open, *v_open;      /* [n_slots][2][kv_heads][QL_KV8_BLOCK][head_dim]; page b of a sequence in [b % 2] */
    const int32_t *page_table;   /* [n_seqs][max_pages] */
    const int32_t *slots;        /* [n_seqs] open rows of each sequence; NULL: sequence s has slot s */
    int32_t n_pages, n_slots, n_seqs, max_pages, kv_heads, head_dim;
} ql_kv8_cache;
/* Rows of a call.  q_start == NULL: row s is the one new token of sequence s (rows == n_seqs).  Otherwise
 * sequence s has rows q_start[s] .. q_start[s + 1] - 1 (q_start[0] = 0, q_start[n_seqs] = rows; none is
 * allowed), at most max_q_len.  kv_len[s] counts the sequence's tokens with this call's among them: its
 * last row has position kv_len[s] - 1.  kv_len[s] == 0: an idle sequence, its row is skipped.
 *
 * ql_kv8_append: per head, q and k are normalised and rotated, k and v stored into the cache.
 *   norm (gamma != NULL): x / sqrt(mean(x^2) + eps) * gamma, gamma [head_dim] f32;
 *   rotation of the first rotary_dim elements (0: none; a multiple of head_dim / 16), pairs (i, i +
 *   rotary_dim / 2) as elsewhere here, by rope [max_positions][rotary_dim] f32 on the device: the cosines
 *   of the position's rotary_dim / 2 angles, then their sines.
 * Row r of q: n_heads heads of head_dim elements from q + r * q_stride (elements), k and v kv_heads heads
 * in the same way, so the stacked output of one projection serves all three; q_out likewise, of the same
 * type, and may be q.  q == NULL (n_heads 0): k and v only.  One launch. */
QL_API int ql_kv8_append(const ql_kv8_cache *cache, int32_t type, const void *q, int64_t q_stride, const void *k,
                         int64_t k_stride, const void *v, int64_t v_stride, void *q_out, int64_t q_out_stride,
                         int n_heads, const float *q_gamma, const float *k_gamma, float eps, const float *rope,
                         int rotary_dim, int max_positions, const int32_t *kv_len, const int32_t *q_start, int rows,
                         int max_q_len);
/* Causal attention of the call's rows over the cache (after ql_kv8_append):
 *   out_h = softmax_j(scale q_h . k_j) . v_j [* sigmoid(gate_h)],  j = 0 .. the row's position,
 * query head h reads KV head h / (n_heads / kv_heads).  gate == NULL: none.  A row that sees no key gets
 * zeros; one that sees a NaN or infinity gets NaN.  Keys and values are read as they stand after the append: a token
 * whose page the same call filled is read as bytes by every row of the call that sees it, while a row that came before
 * the page was full read exact rows.  So the bytes of the cache do not depend on how tokens are cut into calls, but a
 * row's result does, by the quantisation of its own page.
 * f32: fp32 results (1e-6 relative).  q, weights and open rows go through the tensor cores in two f16 limbs, 22 bits (of
 * the row's largest, the weight itself, and the largest of the open page); products are exact, sums fp32.  A weight below
 * 2^-32 of the row's heaviest adds nothing to the values' sum, and the sums take a rounding of at most 2^-24 for every 64
 * keys: one heavy key over n light ones that all agree is right to n 2^-29.  bf16: operands and weights of 16 bits
 * (weights: f16), sums of 32.
 * max_q_len and max_kv_len bound the lengths on the device; the launch, its split over the keys and the choice between
 * the two kernels follow from them, so bounds near the lengths are faster (more cached tokens are read all the same;
 * rows beyond max_q_len are not computed, and reported).  The workspace, ql_kv8_attend_workspace bytes (they depend on
 * head_dim alone: one serves calls of any size, and the largest of several head_dims serves them all), 16-byte aligned,
 * is zeroed by the caller before its first use and left usable by every call; calls that may overlap on the GPU need
 * one each. */
QL_API size_t ql_kv8_attend_workspace(int n_heads, int kv_heads, int head_dim, int n_seqs, int rows, int max_q_len,
                                      int max_kv_len);
QL_API int ql_kv8_attend(const ql_kv8_cache *cache, int32_t type, const void *q, int64_t q_stride, const void *gate,
                         int64_t gate_stride, void *out, int64_t out_stride, int n_heads, float scale,
                         const int32_t *kv_len, const int32_t *q_start, int rows, int max_q_len, int max_kv_len,
                         void *workspace, size_t workspace_bytes);
/* Which kernel this thread's last ql_kv8_attend launched: QL_KV8_FORM_SPLIT (rows of 8, split over the keys),
 * QL_KV8_FORM_TILES (tiles of rows on tcgen05), 0 none.  ctas (nullable): the CTAs that shared the keys of a row. */
#define QL_KV8_FORM_SPLIT 1
#define QL_KV8_FORM_TILES 2
QL_API int ql_kv8_attend_form(int *ctas);
/* The cache's values back: k_out and v_out [n_seqs][count][kv_heads][head_dim] of `type` (either may be
 * NULL), positions start[s] .. start[s] + count - 1 of sequence s (start == NULL: from 0), zeros where the
 * sequence has none.  E.g. to move a sequence to the bf16 cache of ql_full_attention_attend. */
QL_API int ql_kv8_gather(const ql_kv8_cache *cache, int32_t type, void *k_out, void *v_out, const int32_t *start,
                         int count, const int32_t *kv_len);

/* ---- rules on logits (no reference twin; the reference samples from raw logits, Sampler.cpp:24-50) ---
 * Any pointer but history_len and bias_start (which go with history and bias_ids) may be NULL: that rule
 * is off.  All are device pointers. */
typedef struct ql_logits_rules {
    const int32_t *history;      /* [rows][history_stride] token ids: the prompt, then what was generated; */
    int64_t history_stride;      /*   ids outside [0, vocab) are ignored; at most 1048575 ids a row */
    const int32_t *history_len;  /* [rows] */
    const int32_t *prompt_len;   /* [rows] leading ids that are the prompt; NULL: none */
    const float *repetition;     /* [rows] > 0: x / r where x > 0, else x * r, for ids anywhere in the history */
    const float *frequency;      /* [rows]: minus frequency times the number of generated occurrences */
    const float *presence;       /* [rows]: minus presence for generated ids */
    const int32_t *bias_ids;     /* added to ids bias_ids[bias_start[r] .. bias_start[r + 1]); an id listed */
    const float *bias_values;    /*   twice gets both, in list order */
    const int32_t *bias_start;   /* [rows + 1] */
    const uint32_t *mask;        /* [mask_rows][mask_stride] words: bit t % 32 of word t / 32 allows token t, */
    int64_t mask_stride;         /*   0 sets it to -inf */
    int32_t mask_rows;
    const int32_t *mask_row;     /* [rows] mask of each row, < 0: none; NULL: mask r for row r */
} ql_logits_rules;
/* out = the rules applied to logits in the order above, each step rounded once to f32; rows logits_stride
 * and out_stride floats apart; out may be logits (same stride) or NULL.  token (nullable): [rows] the
 * greedy token, lowest id among equals, NaN never; -1 where nothing is above -inf.  With token != NULL the
 * workspace has 16 bytes per row, zeroed by the caller before its first use and left zero by every call. */
QL_API int ql_logits_apply(const float *logits, int64_t logits_stride, float *out, int64_t out_stride, int rows,
                           int vocab, const ql_logits_rules *rules, int32_t *token, void *workspace,
                           size_t workspace_bytes);

/* ---- residual, norm and 8-bit rows (no reference twin as one launch; the reference adds, normalises and quantises in
 *      three, kernel.cu:112-183, 1679-1765) ---------------------------------------------------------------------------
 *   v = x + residual, rounded to `type` (residual == NULL: x);   y = v / sqrt(mean(v^2) + eps) * gamma
 * type: QL_F32 or QL_BF16, of x, residual, sum and y; gamma f32 (NULL: 1).  sum receives v (NULL: not stored) and may be
 * x or residual (same stride); y (NULL: not stored) x or residual.  Strides in elements, at least hidden.
 * xq receives y (before its rounding to type) as Q8_1 rows: layout QL_Q8_ROWS, the bytes that ql_quantize_q8_1 gives
 * for y, rows ql_q8_1_row_bytes(hidden) apart, or QL_Q8_MMQ, those of ql_quantize_q8_1_mmq; QL_Q8_NONE: xq unused.
 * hidden: any up to 32768 (a last block of fewer than 32 is filled with zeros, and the last group of QL_Q8_MMQ with blocks
 * of zeros).  fp32 sums; one launch. */
#define QL_Q8_NONE 0
#define QL_Q8_ROWS 1
#define QL_Q8_MMQ 2
QL_API int ql_add_rms_norm(int32_t type, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                           void *sum, int64_t sum_stride, const float *gamma, float eps, void *y, int64_t y_stride,
                           uint8_t *xq, int layout, int store_raw_sum, int rows, int hidden);

/* ---- choice of experts (ql_moe_router_topk is the reference's: softmax, 64 experts) --------------------------------
 *   s_e = softmax over the token's logits, or 1 / (1 + exp(-logit));   c_e = s_e + bias[e]
 *   n_groups > 1: of n_groups groups of n_experts / n_groups consecutive experts the top_groups best stay, each
 *   counted by the sum of its group_best (1 or 2) largest c;
 *   the k experts of largest c in them, by descending c; equal ones by the lower id (groups likewise);
 *   w_e = s_e [renormalise: / sum of the chosen s, 0 where that is 0] * scale   (the bias is not in the weights)
 * c is compared as 64-bit scores (without a bias, logits); weights are f32 within 2^-18 of the token's largest score (with
 * renormalise of 1) times scale.  A logit that is not finite counts as -inf; such an expert, or one with a bias of -inf or
 * NaN, is never chosen, nor is a group of none but them.  Where fewer than k are left the rest of top_idx is -1 with weight
 * 0 (the grouped experts skip those).  n_experts <= 1024, k <= 32, n_groups <= 32; tokens' rows of logits are logits_stride floats apart. */
#define QL_ROUTE_SOFTMAX 0
#define QL_ROUTE_SIGMOID 1
typedef struct ql_moe_route_rule {
    int32_t score;
    const float *bias; /* device, [n_experts]; NULL: none */
    int32_t n_groups, top_groups, group_best;
    int32_t renormalise;
    float scale;
} ql_moe_route_rule;
QL_API int ql_moe_route(const float *logits, int64_t logits_stride, int32_t *top_idx, float *top_w, int tokens,
                        int n_experts, int k, const ql_moe_route_rule *rule);

/* ---- low-rank adapters beside a shared projection (no reference twin) ----------------------------------------------
 * For rows x of many requests, each with its own adapter i of a pool, beside one to three projections of the same x
 * whose outputs stand side by side in a row of y (q, k and v; gate and up):
 *   h = scale[i] x A_i^T,   y = base + h B_i^T
 * base is what the shared (quantised) projection gave; it may be y (same stride), else it must not overlap y, or NULL for
 * 0.  A row without an adapter gets y = base.  x and y must not overlap.
 * The pool keeps n_adapters slots for each projection, of max_rank ranks; adapter i uses the first rank[i] of them
 * (0: as none), what stands in the rest is not used.  type: QL_F16, QL_BF16 or QL_F32, of A and B.  in_dim: a
 * multiple of 32; max_rank: a multiple of 8 up to 256; out_dim: any.  a and b start on 16 bytes; a pair that is NULL is
 * a projection without adapters.  fp32 results: f16 and bf16 weights enter the tensor cores exactly, f32 ones as two
 * tf32 limbs (22 bits); x and h as three bf16 limbs beside bf16 weights (every bit), else as two limbs (22 bits; h beside
 * f16 weights 22 bits of its row's largest in calls of few rows); sums are fp32.  A row of x that is not finite, or an h
 * that passes fp32's range, gives NaN, in that row alone. */
typedef struct ql_lora_pool {
    int32_t type, n_proj;
    const void *a[3];    /* [n_adapters][max_rank][in_dim] */
    const void *b[3];    /* [n_adapters][out_dim][max_rank] */
    int32_t out_dim[3];  /* outputs of each projection; its first column of y is the sum of those before it */
    int32_t in_dim, n_adapters, max_rank;
    const int32_t *rank; /* device, [n_adapters]; NULL: max_rank */
    const float *scale;  /* device, [n_adapters]; NULL: 1 */
} ql_lora_pool;
/* adapter: device, [n_seqs], the adapter of each sequence, < 0: none.  q_start == NULL: row s is the one row of sequence s
 * (rows == n_seqs); otherwise sequence s has rows q_start[s] .. q_start[s + 1] - 1 (device, [n_seqs + 1], not falling; none is
 * allowed), and rows before the first and behind the last sequence are left as they are.  Both are read on the device, so a
 * captured CUDA graph follows them.  Rows of different sequences with one adapter share its weights.  An adapter outside the
 * pool, or a rank outside 0 .. max_rank, counts as none and is reported by the next ql_check_device (QL_EDEVICE).  One
 * launch; the same call gives the same bits. */
QL_API int ql_lora_add(const ql_lora_pool *pool, const float *x, int64_t x_stride, const float *base, int64_t base_stride,
                       float *y, int64_t y_stride, const int32_t *adapter, int n_seqs, const int32_t *q_start, int rows);
/* Which kernel this thread's last ql_lora_add launched: QL_LORA_FORM_ROWS (tiles of up to 32 rows of an adapter),
 * QL_LORA_FORM_TILES (tiles of 128 rows on tcgen05), 0 none.  ctas (nullable): the CTAs that shared a tile. */
#define QL_LORA_FORM_ROWS 1
#define QL_LORA_FORM_TILES 2
QL_API int ql_lora_add_form(int *ctas);

/* ---- opt-in int8 activation path, Q8_1 (reference kernel.cuh:47-52) -------------------
 * Changes numerics (activations rounded to int8 per 32), as in the reference, which keeps it off
 * by default (TensorTool.cpp:159-161).  Bytes of one Q8_1 row of in_dim activations (36 per 32). */
QL_API size_t ql_q8_1_row_bytes(int in_dim);
/* x [m][in_dim] (rows in_dim apart) -> x_q8_1 [m][ql_q8_1_row_bytes(in_dim)]: per 32 activations
 * f16 d = max|x| / 127, f16 sum (sum of x when store_raw_sum, else d * sum q), 32 int8 q; the same
 * bytes as launch_quantize_q8_1 (launch.cu:201-207). */
QL_API int ql_quantize_q8_1(const float *x, uint8_t *x_q8_1, int in_dim, int m, int store_raw_sum);
/* y[out_dim] = W . x for one Q8_1 activation row: integer dot products per 32-element block with
 * the block scales in fp32 (launch_quant_gemv_q8_1, launch.cu:222-245); Q4_K, Q6_K, Q5_0, Q8_0. */
QL_API int ql_quant_gemv_q8_1(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const uint8_t *x_q8_1,
                              float *y, int out_dim, int in_dim);
/* y[m][out_dim] for m Q8_1 activation rows (ql_q8_1_row_bytes(in_dim) apart), the GEMV's per-block
 * formula for every (token, output row), on the integer tensor cores (launch_quant_matmul_q8_1,
 * launch.cu:512-531); Q4_K, Q6_K, Q5_0, Q8_0. */
QL_API int ql_quant_matmul_q8_1(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const uint8_t *x_q8_1,
                                float *y, int out_dim, int in_dim, int m);
/* The reference's packed (MMQ) Q8_1 layout (kernel.cuh:56-61): 144-byte groups of 4 blocks
 * {4 x (f16 d, f16 sum), 4 x 32 int8}, group-major ([group][row]); ql_q8_1_mmq_row_bytes(in_dim)
 * per row.  The quantizer's bytes equal launch_quantize_q8_1_mmq's; the matmul computes
 * ql_quant_matmul_q8_1's result from that layout (Q4_K, Q6_K, as launch_quant_matmul_q8_1_mmq). */
QL_API size_t ql_q8_1_mmq_row_bytes(int in_dim);
QL_API int ql_quantize_q8_1_mmq(const float *x, uint8_t *x_q8_1_mmq, int in_dim, int m, int store_raw_sum);
QL_API int ql_quant_matmul_q8_1_mmq(int32_t quant_type, const uint8_t *weight, size_t row_bytes,
                                    const uint8_t *x_q8_1_mmq, float *y, int out_dim, int in_dim, int m);

/* ---- embedding, dequant, argmax (reference kernel.cuh:141-142, 244-253, 347) ----- */
QL_API int ql_quant_embedding(int32_t quant_type, const int *input, float *output, const uint8_t *table, size_t row_bytes,
                       int hidden_size, int input_size);
/* Whole-tensor dequant to IEEE f16 bits, num_elements a multiple of the block size. */
QL_API int ql_dequantize_to_f16(int32_t quant_type, const uint8_t *src, uint16_t *out, int64_t num_elements);
QL_API int ql_dequantize_q4k_to_f16(const uint8_t *src, uint16_t *out, int64_t num_elements);
QL_API int ql_dequantize_q80_to_f16(const uint8_t *src, uint16_t *out, int64_t num_elements);
QL_API int ql_dequantize_q50_to_f16(const uint8_t *src, uint16_t *out, int64_t num_elements);
QL_API int ql_dequantize_q6k_to_f16(const uint8_t *src, uint16_t *out, int64_t num_elements);
QL_API int ql_dequantize_q40_to_f16(const uint8_t *src, uint16_t *out, int64_t num_elements);
/* out_idx[0] = argmax(logits[0..n)), lowest index on ties. */
QL_API int ql_argmax(const float *logits, int n, int *out_idx);

/* Same result as ql_argmax, without ever allocating device memory.  No
 * counterpart in the reference.  For callers that cannot let a library call
 * cudaMalloc: a server whose HBM is owned by its own pool or budgeted once at
 * start-up (weights, KV cache), or code under an allocation ban after start-up.
 * The partials live in a fixed 8 KB array inside the library's device image: n
 * is limited to 16,777,216 (larger n returns QL_EINVAL); calls that overlap on
 * the GPU race on the shared array; the first call on a device performs a
 * one-time set-up (resolving the array's address) and should come before any
 * stream capture; do not use it on a device after cudaDeviceReset. */
QL_API int ql_argmax_noalloc(const float *logits, int n, int *out_idx);

/* ---- fused forms (no reference counterpart; fusions the reference runs as
 *      separate rms_norm / add kernels, kernel.cu:80-84,112-147) ------------------ */
/* y[m*y_stride + o] (=|+=) W[o] . rmsnorm(x[m*x_stride + :]) (+ bias[o]).
 * norm_gamma == NULL skips the norm; bias may be NULL; accumulate != 0 adds into y. */
QL_API int ql_quant_gemv_ex(int32_t quant_type, const uint8_t *weight, size_t row_bytes, const float *x, int64_t x_stride,
                     float *y, int64_t y_stride, int out_dim, int in_dim, int m, const float *norm_gamma, float eps,
                     const float *bias, int accumulate);
/* Fused projections sharing one activation (e.g. q, k and v): the outputs of
 * nsrc (1..3) matrices, stacked by rows, y[m*y_stride + r] for r < sum(rows),
 * with one optional RMSNorm and a stacked bias.  Every source but the last must
 * have a multiple of 32 rows.  w, row_bytes and rows are host arrays of nsrc. */
QL_API int ql_quant_gemv_stacked_ex(int32_t quant_type, int nsrc, const uint8_t *const *weights,
                                    const size_t *row_bytes, const int *rows, const float *x, int64_t x_stride,
                                    float *y, int64_t y_stride, int in_dim, int m, const float *norm_gamma, float eps,
                                    const float *bias);
/* act[m*act_stride + f] = SiLU(Wg[f] . n(x_m)) * (Wu[f] . n(x_m)), n = optional RMSNorm. */
QL_API int ql_quant_swiglu_ex(int32_t quant_type, const uint8_t *gate_weight, const uint8_t *up_weight,
                       size_t gate_row_bytes, size_t up_row_bytes, const float *x, int64_t x_stride, float *act,
                       int64_t act_stride, int ffn_dim, int in_dim, int m, const float *norm_gamma, float eps);
/* y = x * rsqrt(mean(x^2) + eps) * gamma (gamma f32, may be NULL), rows x hidden. */
QL_API int ql_rms_norm_f32(const float *x, float *y, const float *gamma, int rows, int hidden, float eps);

/* ---- GGUF loader (reference GgufFile, src/format/gguf/GgufFile.cpp:152-250, and
 *      MF::validate, src/format/MF.cpp:43-84) --------------------------------------
 * ql_gguf_open maps a GGUF v2/v3 file read-only and parses its metadata and tensor table
 * (QL_EINVAL with a message on any format error; every length is checked against the file).
 * Tensor shapes are reported outermost-first (the file stores dims innermost-first); data
 * points into the mapping (host memory, valid until ql_gguf_close); nbytes follows the ggml
 * block traits.  The data section starts at the end of the tensor table rounded up to
 * general.alignment (default 32).  ql_gguf_find_tensor returns the index or -1.
 * ql_gguf_metadata_type returns the GGUF value type (0..12) or -1 when the key is absent;
 * integer, bool and float values convert between the int and float getters.
 * ql_gguf_validate applies MF::validate's container checks (tensors present, names non-empty
 * and unique, shapes non-empty with positive dims, data present) and admits the types this
 * library computes with: F32, F16, BF16, Q4_0, Q4_K, Q5_0, Q6_K, Q8_0 (the reference's
 * validator leaves Q4_0 out although its parser reads it). */
QL_API int ql_gguf_open(const char *path, void **file);
QL_API int ql_gguf_close(void *file);
QL_API int ql_gguf_version(void *file);
QL_API int64_t ql_gguf_tensor_count(void *file);
QL_API int64_t ql_gguf_find_tensor(void *file, const char *name);
QL_API int ql_gguf_tensor_info(void *file, int64_t index, const char **name, int32_t *quant_type, int32_t *n_dims,
                               int64_t *shape /* [8] */, const uint8_t **data, size_t *nbytes);
QL_API int ql_gguf_metadata_type(void *file, const char *key);
QL_API int ql_gguf_metadata_int(void *file, const char *key, int64_t *out);
QL_API int ql_gguf_metadata_float(void *file, const char *key, double *out);
QL_API int ql_gguf_metadata_string(void *file, const char *key, const char **out);
QL_API int64_t ql_gguf_metadata_array_len(void *file, const char *key);
QL_API int ql_gguf_metadata_array_int(void *file, const char *key, int64_t index, int64_t *out);
QL_API int ql_gguf_metadata_array_float(void *file, const char *key, int64_t index, double *out);
QL_API int ql_gguf_metadata_array_string(void *file, const char *key, int64_t index, const char **out);
QL_API int ql_gguf_validate(void *file);
/* Weight upload (reference CudaWeightPool::cached_weight, CudaWeightPool.cpp:119-175, which
 * uploads the raw blocks unchanged): copies rows [row0, row0 + nrows) of a host matrix whose
 * rows are row_bytes apart, bytes [byte0, byte0 + nbytes_per_row) of each row, to dst (device,
 * rows packed nbytes_per_row apart), as one pitched copy on the current stream.  A whole matrix
 * is byte0 = 0, nbytes_per_row = row_bytes; a column-parallel shard a row range; a row-parallel
 * shard whole blocks of every row (byte0 and nbytes_per_row multiples of the block bytes).  The
 * kernels read the raw GGUF layout, so no repack is needed.  Pinned host memory makes the copy
 * asynchronous; pageable memory makes it synchronous. */
QL_API int ql_weight_upload(const uint8_t *host, size_t row_bytes, int64_t row0, int64_t nrows, size_t byte0,
                            size_t nbytes_per_row, uint8_t *dst);

/* ---- synthetic weights (benchmarks; no reference counterpart) -------------------- */
/* dst[rows x row_bytes] = quantize(N(0, std) with seed), generated on the device. */
QL_API int ql_synth_quantized(int32_t quant_type, uint64_t seed, int64_t rows, int in_dim, float std, uint8_t *dst);

/* ---- introspection ------------------------------------------------------------- */
/* Bytes per row of `in_dim` elements of `quant_type` (0 if not a block multiple). */
QL_API size_t ql_row_bytes(int32_t quant_type, int in_dim);
/* Number of kernel launches the last call on this thread issued. */
QL_API int ql_last_launch_count(void);

#ifdef __cplusplus
}
#endif

#endif /* QLINEAR_B200_H */
