/*
 * tecoops.h — C ABI of the MI355X (gfx950) LLM-inference operator library.
 *
 * Drop-in for the reference interface teco/interface/include/tecoops.h:37-188.
 * Every enum value, handle/descriptor function and op signature of the
 * reference is kept; the only type change is the stream: sdaaStream_t
 * (reference tecoops.h:92-93) becomes hipStream_t.  All tensors are device
 * pointers owned by the caller; every entry point validates its arguments
 * before any device work, enqueues on the handle's stream and returns without
 * synchronising.
 *
 * Entry points below the "Extensions" banner have no counterpart in the
 * reference header.  They are additive: bf16 through a dataType argument,
 * rotary embedding, GEMV (fp16 / int8 weights), causal_conv1d with bias and
 * arbitrary strides, flash attention with cumulative query offsets and an
 * explicit softmax scale.
 */
#ifndef TECOOPS_INCLUDE_TECOOPS_H_
#define TECOOPS_INCLUDE_TECOOPS_H_

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* reference tecoops.h:37 */
#define TECOOPS_DIM_MAX 8

/* reference tecoops.h:39-47 — values are part of the ABI. */
typedef enum {
    TECOOPS_STATUS_SUCCESS = 0,
    TECOOPS_STATUS_NOT_INITIALIZED = 1,
    TECOOPS_STATUS_ALLOC_FAILED = 2,
    TECOOPS_STATUS_BAD_PARAM = 3,
    TECOOPS_STATUS_INTERNAL_ERROR = 4,
    TECOOPS_STATUS_INVALID_VALUE = 5,
    TECOOPS_STATUS_NOT_SUPPORTED = 6,
} tecoopsStatus_t;

/* reference tecoops.h:49-58 */
typedef enum {
    TECOOPS_TENSOR_NCHW = 0,
    TECOOPS_TENSOR_NHWC = 1,
    TECOOPS_TENSOR_CHWN = 2,
    TECOOPS_TENSOR_NWHC = 3,
    TECOOPS_TENSOR_NCDHW = 4,
    TECOOPS_TENSOR_NDHWC = 5,
    TECOOPS_TENSOR_CDHWN = 6,
} tecoopsTensorFormat_t;

/* reference tecoops.h:60-71 */
typedef enum {
    TECOOPS_ALGO_0 = 0,
    TECOOPS_ALGO_1,
    TECOOPS_ALGO_2,
    TECOOPS_ALGO_3,
    TECOOPS_ALGO_4,
    TECOOPS_ALGO_5,
    TECOOPS_ALGO_6,
    TECOOPS_ALGO_7,
    TECOOPS_ALGO_8,
    TECOOPS_ALGO_9,
} tecoopsAlgo_t;

/* reference tecoops.h:73-85 */
typedef enum {
    TECOOPS_DATA_FLOAT = 0,
    TECOOPS_DATA_HALF = 1,
    TECOOPS_DATA_INT8 = 2,
    TECOOPS_DATA_INT16 = 3,
    TECOOPS_DATA_INT32 = 4,
    TECOOPS_DATA_INT64 = 5,
    TECOOPS_DATA_UINT8 = 6,
    TECOOPS_DATA_BOOL = 7,
    TECOOPS_DATA_DOUBLE = 8,
    TECOOPS_DATA_BFLOAT16 = 9,
    TECOOPS_DATA_COMPLEX_FLOAT = 10,
} tecoopsDataType_t;

/* reference tecoops.h:87-88 */
typedef struct tecoopsContext *tecoopsHandle_t;
typedef struct tecoopsTensorStruct *tecoopsTensorDescriptor_t;

/* ---- handle (reference tecoops.h:90-94; impl tecoops.cpp:38-68, :239-258) ---- */
tecoopsStatus_t tecoopsCreate(tecoopsHandle_t *handle);
tecoopsStatus_t tecoopsDestroy(tecoopsHandle_t handle);
tecoopsStatus_t tecoopsSetStream(tecoopsHandle_t handle, hipStream_t stream);
tecoopsStatus_t tecoopsGetStream(tecoopsHandle_t handle, hipStream_t *stream);
const char *tecoopsGetErrorString(tecoopsStatus_t status);

/* ---- tensor descriptors (reference tecoops.h:96-123; impl tecoops.cpp:70-237) ---- */
tecoopsStatus_t tecoopsCreateTensorDescriptor(tecoopsTensorDescriptor_t *tensorDesc);
tecoopsStatus_t tecoopsSetTensor4dDescriptor(tecoopsTensorDescriptor_t tensorDesc,
                                             tecoopsTensorFormat_t format,
                                             tecoopsDataType_t dataType,
                                             int n, int c, int h, int w);
tecoopsStatus_t tecoopsGetTensor4dDescriptor(const tecoopsTensorDescriptor_t tensorDesc,
                                             tecoopsDataType_t *dataType,
                                             int *n, int *c, int *h, int *w,
                                             int *nStride, int *cStride, int *hStride,
                                             int *wStride);
tecoopsStatus_t tecoopsSetTensorNdDescriptor(tecoopsTensorDescriptor_t tensorDesc,
                                             tecoopsDataType_t dataType, int nbDims,
                                             const int dimA[], const int strideA[]);
tecoopsStatus_t tecoopsGetTensorNdDescriptor(const tecoopsTensorDescriptor_t tensorDesc,
                                             int nbDimsRequested, tecoopsDataType_t *dataType,
                                             int *nbDims, int dimA[], int strideA[]);
tecoopsStatus_t tecoopsDestroyTensorDescriptor(tecoopsTensorDescriptor_t tensorDesc);

/* ---- ops outside the LLM path (reference tecoops.h:125-126, :139-145).
 *      Exported for ABI completeness; they return TECOOPS_STATUS_NOT_SUPPORTED
 *      after argument validation. ---- */
tecoopsStatus_t tecoopsFlattenRays(tecoopsHandle_t handle, const int *rays, uint32_t N, uint32_t M,
                                   int *res, tecoopsAlgo_t algo);
tecoopsStatus_t tecoopsReduceVariance(const tecoopsHandle_t handle, int axis, int correction,
                                      const tecoopsTensorDescriptor_t xDesc, const void *x,
                                      const tecoopsTensorDescriptor_t yDesc, void *y);
tecoopsStatus_t tecoopsMorton3DInvert(tecoopsHandle_t handle, const int *indices, uint32_t N,
                                      int *coords);

/* ---- memset (reference tecoops.h:128; impl ops/memset.cpp:52-67).
 *      Fills `size` bytes at x with (uint8_t)value. ---- */
tecoopsStatus_t tecoopsMemset(tecoopsHandle_t handle, void *x, const int value, size_t size);

/* ---- reshape_and_cache (reference tecoops.h:130-137; impl ops/reshape_and_cache.cpp:64-105).
 *      key/value fp16 [num_tokens, num_kv_heads, head_size];
 *      caches fp16 [num_blocks, num_kv_heads, block_size, head_size];
 *      slot_mapping int64 [num_tokens]; slot < 0 is skipped.  Slots at or beyond
 *      num_blocks*block_size are also skipped (the reference would write out of
 *      bounds there). ---- */
tecoopsStatus_t tecoopsReshapeAndCache(tecoopsHandle_t handle,
                                       const void *key, const void *value,
                                       const int64_t *slot_mapping,
                                       void *key_cache, void *value_cache,
                                       int num_tokens, int num_kv_heads, int head_size,
                                       int num_blocks, int block_size);

/* ---- rms_norm (reference tecoops.h:147-156; impl ops/rms_norm.cpp:64-100).
 *      fp16 [num_tokens, hidden_size].  residual != NULL selects the fused
 *      add variant and then requires residual_out. ---- */
tecoopsStatus_t tecoopsRmsNorm(tecoopsHandle_t handle,
                               const void *input, const void *weight, const void *residual,
                               void *output, void *residual_out,
                               int num_tokens, int hidden_size, float eps);

/* ---- flash_attention (reference tecoops.h:158-169; impl ops/flash_attention.cpp:71-119).
 *      Paged, varlen, bottom-right causal, GQA.  q [sum(q_seq_lens), H, D];
 *      caches [num_blocks, Hkv, block_size, D]; blockTable int32
 *      [batch, max_blocks_per_seq]; q_seq_lens / kv_seq_lens int32 [batch]
 *      (device).  Scale is 1/sqrt(D).  Element type comes from the
 *      descriptors: TECOOPS_DATA_HALF or TECOOPS_DATA_BFLOAT16 (q, caches and
 *      output must agree).  D in {32, 64, 96, 128, 160, 192}; any
 *      block_size >= 1.  As in the reference, the results do not depend on
 *      max_seqlen_q / max_seqlen_k (any value, also <= 0, is accepted): they
 *      only shape the launch, and a bound that holds makes it fastest.
 *      kv lengths past block_table_dim * block_size (the reference's
 *      precondition) are clamped to it.  max_block_num and workspace are
 *      accepted and ignored, as in the reference (flash_attention.cpp:110):
 *      the split-KV partials of decode live in the handle's scratch, one
 *      buffer per stream the handle runs on. ---- */
tecoopsStatus_t tecoopsFlashAttention(tecoopsHandle_t handle,
                                      int max_seqlen_q, int max_seqlen_k,
                                      int max_block_num, const int *q_seq_lens,
                                      const int *kv_seq_lens,
                                      const tecoopsTensorDescriptor_t blockTableDesc,
                                      const void *blockTable,
                                      const tecoopsTensorDescriptor_t qDataDesc,
                                      const void *qData,
                                      const tecoopsTensorDescriptor_t kCacheDesc,
                                      const void *kCache,
                                      const tecoopsTensorDescriptor_t vCacheDesc,
                                      const void *vCache,
                                      const tecoopsTensorDescriptor_t oDataDesc,
                                      void *oData, void *workspace);

/* ---- causal_conv1d (reference tecoops.h:171-188; impl ops/causal_conv1d.cpp:56-105).
 *      x/out fp16 [totalSeqLen, dim] with token strides xSeqStride/outSeqStride;
 *      weight fp16 [width, dim]; convState fp16 [entries, width-1, dim] with
 *      entry stride convStateStride.  SiLU is always applied (actMode is
 *      ignored, as in the reference).  queryStartLoc NULL means one token per
 *      sequence; convStateIndices NULL means the identity. width in [2, 4]. ---- */
tecoopsStatus_t tecoopsCausalConv1d(tecoopsHandle_t handle,
                                    int batch, int totalSeqLen, int dim, int width,
                                    int convStateStride, int xSeqStride, int outSeqStride,
                                    int padSlotId, int api_mode, int actMode,
                                    const void *x, void *convState, const void *weight,
                                    void *out,
                                    const int *queryStartLoc,
                                    const int *convStateIndices,
                                    const int8_t *hasInitialState);

/* ======================== Extensions (no reference counterpart) ======================== */

/* rms_norm with an explicit element type (TECOOPS_DATA_HALF or
 * TECOOPS_DATA_BFLOAT16); otherwise identical to tecoopsRmsNorm. */
tecoopsStatus_t tecoopsRmsNormEx(tecoopsHandle_t handle,
                                 const void *input, const void *weight, const void *residual,
                                 void *output, void *residual_out,
                                 int num_tokens, int hidden_size, float eps,
                                 tecoopsDataType_t dataType);

/* reshape_and_cache for any 2-byte element type (HALF / BFLOAT16): the copy is
 * bit-exact, so only the element size matters. */
tecoopsStatus_t tecoopsReshapeAndCacheEx(tecoopsHandle_t handle,
                                         const void *key, const void *value,
                                         const int64_t *slot_mapping,
                                         void *key_cache, void *value_cache,
                                         int num_tokens, int num_kv_heads, int head_size,
                                         int num_blocks, int block_size,
                                         tecoopsDataType_t dataType);

/* Flash attention with the arguments the reference's torch wrapper accepts but
 * drops (api/torch_ext.cpp:99-165): cu_seqlens_q int32 [batch+1] (device) is
 * used when q_seq_lens is NULL, so callers need no host synchronisation;
 * softmax_scale > 0 overrides 1/sqrt(D); causal = 0 disables the mask.
 * With cu_seqlens_q, output rows past cu_seqlens_q[batch] (rows of no
 * sequence, e.g. a graph's padding) are written as zeros, as the reference
 * torch wrapper zeroes its output first (api/torch_ext.cpp:128-132).
 * workspace NULL uses the handle's scratch for a split-KV decode; on a stream
 * being captured into a graph that call returns TECOOPS_STATUS_NOT_SUPPORTED
 * (a later call may free the scratch the graph would keep): pass a workspace
 * or call tecoopsFlashAttentionNoAlloc there.  A workspace must hold
 * tecoopsGetFlashAttentionWorkspaceSize() bytes for the same batch, heads,
 * head size, max_seqlen_q and max_seqlen_k, and max_seqlen_k must then be > 0
 * (it sizes the split-KV partials).  A prefill without a workspace whose
 * longest context outweighs the rest (chunks of prompts over cached context)
 * splits its keys too, in up to 98 MiB of the handle's scratch per stream;
 * under capture, on more streams than the handle keeps scratch for, or where no
 * memory is free it runs unsplit, to the same results up to rounding. */
tecoopsStatus_t tecoopsFlashAttentionEx(tecoopsHandle_t handle,
                                        int max_seqlen_q, int max_seqlen_k,
                                        const int *q_seq_lens, const int *cu_seqlens_q,
                                        const int *kv_seq_lens,
                                        const tecoopsTensorDescriptor_t blockTableDesc,
                                        const void *blockTable,
                                        const tecoopsTensorDescriptor_t qDataDesc,
                                        const void *qData,
                                        const tecoopsTensorDescriptor_t kCacheDesc,
                                        const void *kCache,
                                        const tecoopsTensorDescriptor_t vCacheDesc,
                                        const void *vCache,
                                        const tecoopsTensorDescriptor_t oDataDesc,
                                        void *oData, float softmax_scale, int causal,
                                        void *workspace);

/* Flash attention that allocates nothing, for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  No counterpart in the reference.  Arguments and
 * results are those of tecoopsFlashAttentionEx without a workspace (a prefill
 * that it splits runs unsplit here, which rounds differently): the split-KV
 * partials of decode go to a static device array of 64 MiB per GPU (held until
 * the process ends) instead of the handle's scratch, and a call whose decode
 * plan needs more returns TECOOPS_STATUS_BAD_PARAM.  Every call on a GPU
 * shares that array: calls that overlap on one GPU (different streams, threads
 * or handles) race and must be ordered by the caller. */
tecoopsStatus_t tecoopsFlashAttentionNoAlloc(tecoopsHandle_t handle,
                                             int max_seqlen_q, int max_seqlen_k,
                                             const int *q_seq_lens, const int *cu_seqlens_q,
                                             const int *kv_seq_lens,
                                             const tecoopsTensorDescriptor_t blockTableDesc,
                                             const void *blockTable,
                                             const tecoopsTensorDescriptor_t qDataDesc,
                                             const void *qData,
                                             const tecoopsTensorDescriptor_t kCacheDesc,
                                             const void *kCache,
                                             const tecoopsTensorDescriptor_t vCacheDesc,
                                             const void *vCache,
                                             const tecoopsTensorDescriptor_t oDataDesc,
                                             void *oData, float softmax_scale, int causal);

/* Bytes of caller workspace tecoopsFlashAttentionEx needs for these sizes
 * (max_seqlen_k > 0; max_seqlen_q <= 0 sizes for the longest q length the
 * split-KV decode route takes). */
tecoopsStatus_t tecoopsGetFlashAttentionWorkspaceSize(int batch, int num_heads,
                                                      int head_size, int max_seqlen_q,
                                                      int max_seqlen_k, size_t *bytes);

/* causal_conv1d with bias and general strides.
 *   element (b, t, d) of x lives at
 *     x + b*xBatchStride + t*xSeqStride + d*xDimStride     when queryStartLoc == NULL
 *     x + (queryStartLoc[b] + t)*xSeqStride + d*xDimStride  otherwise;
 *   out likewise.  With queryStartLoc == NULL every sequence has seqLen tokens.
 *   weight element (d, k) at weight + d*wDimStride + k*wWidthStride.
 *   bias fp16 [dim] or NULL; silu != 0 applies SiLU.  State semantics are
 *   those of tecoopsCausalConv1d.  The [batch, dim, seqlen] layout of
 *   BASELINE-style callers is xBatchStride = dim*seqlen, xDimStride = seqlen,
 *   xSeqStride = 1. */
tecoopsStatus_t tecoopsCausalConv1dEx(tecoopsHandle_t handle,
                                      int batch, int seqLen, int dim, int width,
                                      const void *x, long long xBatchStride,
                                      long long xSeqStride, long long xDimStride,
                                      void *out, long long outBatchStride,
                                      long long outSeqStride, long long outDimStride,
                                      const void *weight, int wDimStride, int wWidthStride,
                                      const void *bias,
                                      void *convState, int convStateStride,
                                      const int *queryStartLoc,
                                      const int *convStateIndices,
                                      const int8_t *hasInitialState,
                                      int padSlotId, int api_mode, int silu);

/* Rotary position embedding, in place on query [num_tokens, num_heads, head_size]
 * and key [num_tokens, num_kv_heads, head_size] (token strides query_stride /
 * key_stride in elements; key may be NULL).  The first rot_dim dims of each
 * head rotate by theta_i = pos * base^(-2i/rot_dim), i < rot_dim/2.
 * is_neox != 0 pairs (i, i + rot_dim/2); otherwise (2i, 2i+1).
 * cos_sin_cache (float32 [max_position, rot_dim]: cos then sin) may be NULL,
 * in which case the angles are computed from base.  dataType HALF or
 * BFLOAT16.  Positions outside [0, max_position) with a cache are skipped. */
tecoopsStatus_t tecoopsRotaryEmbedding(tecoopsHandle_t handle, const int64_t *positions,
                                       void *query, void *key,
                                       int num_tokens, int num_heads, int num_kv_heads,
                                       int head_size, int rot_dim,
                                       long long query_stride, long long key_stride,
                                       const float *cos_sin_cache, int max_position,
                                       float base, int is_neox, tecoopsDataType_t dataType);

/* Fused decode step over the paged KV cache: rotary embedding on query (in
 * place) and key as tecoopsRotaryEmbedding, then the rotated key and value
 * [num_tokens, num_kv_heads, head_size] (token stride value_stride) stored at
 * slot_mapping[t] of key_cache / value_cache [num_blocks, num_kv_heads,
 * block_size, head_size] as tecoopsReshapeAndCache (slots < 0 or past the
 * cache are not stored).  write_key != 0 also writes the rotated key back in
 * place.  The cached values are bit-identical to those two calls in sequence. */
tecoopsStatus_t tecoopsRotaryReshapeAndCache(tecoopsHandle_t handle, const int64_t *positions,
                                             void *query, void *key, const void *value,
                                             const int64_t *slot_mapping,
                                             void *key_cache, void *value_cache,
                                             int num_tokens, int num_heads, int num_kv_heads,
                                             int head_size, int rot_dim,
                                             long long query_stride, long long key_stride,
                                             long long value_stride,
                                             const float *cos_sin_cache, int max_position,
                                             float base, int is_neox,
                                             int num_blocks, int block_size, int write_key,
                                             tecoopsDataType_t dataType);

/* y[b, n] = sum_k W[n, k] * x[b, k], fp32 accumulation.
 * W [n, k] row-major, x [batch, k], y [batch, n]; dataType HALF or BFLOAT16. */
tecoopsStatus_t tecoopsGemv(tecoopsHandle_t handle, const void *weight, const void *x, void *y,
                            int batch, int n, int k, tecoopsDataType_t dataType);

/* y[b, n] = scales[n] * sum_k float(Wq[n, k]) * x[b, k], fp32 accumulation.
 * Wq int8 [n, k] row-major, scales fp16 [n], x / y fp16. */
tecoopsStatus_t tecoopsGemvInt8(tecoopsHandle_t handle, const int8_t *weight,
                                const void *scales, const void *x, void *y,
                                int batch, int n, int k);

/* ---- operators of a decoder layer around attention ---- */

typedef enum {
    TECOOPS_ACTIVATION_NONE = 0,
    TECOOPS_ACTIVATION_RELU = 1,
    TECOOPS_ACTIVATION_SILU = 2,
    TECOOPS_ACTIVATION_GELU = 3,      /* v Phi(v) */
    TECOOPS_ACTIVATION_GELU_TANH = 4, /* its tanh form */
} tecoopsActivation_t;

/* Matrix product with its epilogue, fp32 accumulation and one rounding:
 *   out[m, n] = act(sum_k x[m, k] W[n, k] + bias[n]) + residual[m, n].
 * gated != 0: weight holds n gate rows, then n up rows, bias [2n] likewise, and
 *   out[m, n] = act(gate[m, n]) * up[m, n] + residual[m, n].
 * x [m, k], residual and out [m, n] with row strides in elements (elements of a
 * row adjacent); weight [n or 2n, k] packed; bias and residual may be NULL.
 * residual may be out itself (same pointer and stride); other overlaps of out
 * with an input are not allowed.  dataType HALF or BFLOAT16, any sizes (rows
 * of x and W in whole, aligned 16-byte words are fastest) up to k and x_stride
 * 2^21, n 2^23 and 2^23 tiles of out; m = 0 is done without a launch.
 * workspace: tecoopsGetLinearWorkspaceSize() bytes for the same sizes let few
 * tiles be split along k, wherever x and weight lie; with less, or NULL, the call runs with fewer splits
 * (slower, the same result up to fp32 rounding).  Nothing is allocated. */
tecoopsStatus_t tecoopsLinear(tecoopsHandle_t handle, const void *x, long long x_stride,
                              const void *weight, const void *bias,
                              const void *residual, long long residual_stride,
                              void *out, long long out_stride, int m, int n, int k,
                              tecoopsActivation_t activation, int gated,
                              void *workspace, size_t workspace_bytes,
                              tecoopsDataType_t dataType);
tecoopsStatus_t tecoopsGetLinearWorkspaceSize(int m, int n, int k, int gated, size_t *bytes);

/* Mixture-of-experts layer.  Per token t with p = softmax(router_logits[t]):
 *   the top_k experts e_j of the largest logits (ties to the lowest index; -inf
 *   and NaN are never chosen, so a masked token may have fewer or none),
 *   w_j = p[e_j], divided by their sum when renormalize != 0,
 *   h_j = act(x[t] Wg[e_j]^T) * (x[t] Wu[e_j]^T), held to 16 bits or more of
 *         its mantissa (fp16 22; there infinite from 65520 * 256 on),
 *   out[t] = sum_j w_j (h_j W_out[e_j]^T), fp32 sums, one rounding.
 * x [tokens, hidden] with row stride x_stride (elements); w_in [experts,
 * 2 inter, hidden] packed, the inter gate rows Wg of an expert before its up
 * rows Wu; w_out [experts, hidden, inter] packed; router_logits [tokens,
 * experts] packed, logitsType FLOAT or dataType; out [tokens, hidden] packed,
 * zero for a token without experts; out must not overlap an input.  topk_ids
 * int32 and topk_weights float [tokens, top_k] are written unless NULL, best
 * first, -1 and 0 where there is none.  For decode batches: an expert's weights
 * are read once for up to 4, 8 or 16 of its tokens (batches of that many), 16, 32 or
 * 64 (larger ones, by their mean per expert), and again for every 512 tokens of the
 * batch; a prompt, or most tokens at few experts, reads them many times.  Up to 2^30
 * tokens, 1024 experts, top_k 32, hidden and inter 2^16; hidden, inter and
 * x_stride multiples of 8 and 16-byte aligned tensors are fast; tokens = 0 is done
 * without a launch.
 * workspace: tecoopsGetMoeLayerWorkspaceSize() bytes, 16-byte aligned; NULL
 * uses the handle's scratch (NOT_SUPPORTED on a stream under capture). */
tecoopsStatus_t tecoopsMoeLayer(tecoopsHandle_t handle, const void *x, long long x_stride,
                                const void *w_in, const void *w_out, const void *router_logits,
                                tecoopsDataType_t logitsType, void *out, int *topk_ids,
                                float *topk_weights, int tokens, int hidden, int inter,
                                int experts, int top_k, int renormalize,
                                tecoopsActivation_t activation, void *workspace,
                                size_t workspace_bytes, tecoopsDataType_t dataType);
tecoopsStatus_t tecoopsGetMoeLayerWorkspaceSize(int tokens, int hidden, int inter, int experts,
                                                int top_k, size_t *bytes);

/* Rotary positions of several axes (time, height, width of images and video).
 * As tecoopsRotaryEmbedding, but positions is int64 [axes, num_tokens] (rows
 * position_stride elements apart, at least num_tokens, or 0: all axes at the same
 * positions, as in plain text) and pair i of a head turns by the position of one
 * axis.  sections (host, [axes]) are the axes'
 * numbers of frequencies; their sum has to be rot_dim / 2.
 *   CONTIGUOUS   the first sections[0] pairs to axis 0, the next to axis 1, ...;
 *                pair i at base^(-2i/rot_dim)
 *   INTERLEAVED  pair i to axis a = i % axes while i < axes * sections[a], else
 *                to axis 0; pair i at base^(-2i/rot_dim).  The last pair of each
 *                axis but the first has to lie within rot_dim / 2.
 *   PER_AXIS     in ranges as CONTIGUOUS, but the j-th of an axis' n pairs at
 *                base^(-j/n)
 * With a cos_sin_cache (float32 [max_position, rot_dim]) column i of either half
 * is pair i; a token with any position outside it is left as it is.  Without,
 * angles are computed in 64 bits from base as given, a float. */
#define TECOOPS_ROTARY_MAX_AXES 4
typedef enum {
    TECOOPS_ROTARY_CONTIGUOUS = 0,
    TECOOPS_ROTARY_INTERLEAVED = 1,
    TECOOPS_ROTARY_PER_AXIS = 2,
} tecoopsRotaryLayout_t;

tecoopsStatus_t tecoopsRotaryEmbeddingAxes(tecoopsHandle_t handle, const int64_t *positions,
                                           long long position_stride, int axes,
                                           const int *sections, tecoopsRotaryLayout_t layout,
                                           void *query, void *key, int num_tokens, int num_heads,
                                           int num_kv_heads, int head_size, int rot_dim,
                                           long long query_stride, long long key_stride,
                                           const float *cos_sin_cache, int max_position,
                                           float base, int is_neox, tecoopsDataType_t dataType);

/* The same fused with the store into the paged caches, as
 * tecoopsRotaryReshapeAndCache; the cached values are bit-identical to the two
 * calls in sequence. */
tecoopsStatus_t tecoopsRotaryAxesReshapeAndCache(tecoopsHandle_t handle, const int64_t *positions,
                                                 long long position_stride, int axes,
                                                 const int *sections,
                                                 tecoopsRotaryLayout_t layout, void *query,
                                                 void *key, const void *value,
                                                 const int64_t *slot_mapping, void *key_cache,
                                                 void *value_cache, int num_tokens, int num_heads,
                                                 int num_kv_heads, int head_size, int rot_dim,
                                                 long long query_stride, long long key_stride,
                                                 long long value_stride,
                                                 const float *cos_sin_cache, int max_position,
                                                 float base, int is_neox, int num_blocks,
                                                 int block_size, int write_key,
                                                 tecoopsDataType_t dataType);

/* ---- a decode path held in 4 bits: norms with the rotation, the cache, its
 *      attention, weight products ---- */

/* The norm of each head of query and key, then the rotation, in one pass, in
 * place:  y = x / sqrt(mean(x^2) + eps) * w over the head_size elements of a head
 * (w: query_weight or key_weight, [head_size] of dataType), then y turned as
 * tecoopsRotaryEmbeddingAxes turns it; fp32 throughout, one rounding.  key may be
 * NULL, with key_weight.  Positions, sections and layout are those of
 * tecoopsRotaryEmbeddingAxes; sections may be NULL for one axis.  A token with a
 * position outside the cos_sin_cache is left as it is, not normalised either.
 * head_size up to 1024, fewer than 2^24 tokens, up to 2^20 heads a token (head sizes in
 * whole 16-byte words, aligned, up to 512 are fastest; others up to 2^25 heads of all
 * tokens). */
tecoopsStatus_t tecoopsQkNormRotary(tecoopsHandle_t handle, const int64_t *positions,
                                    long long position_stride, int axes, const int *sections,
                                    tecoopsRotaryLayout_t layout, void *query, void *key,
                                    const void *query_weight, const void *key_weight, float eps,
                                    int num_tokens, int num_heads, int num_kv_heads, int head_size,
                                    int rot_dim, long long query_stride, long long key_stride,
                                    const float *cos_sin_cache, int max_position, float base,
                                    int is_neox, tecoopsDataType_t dataType);

/* The same fused with the store into the paged caches, as
 * tecoopsRotaryReshapeAndCache: the cached values are bit-identical to the two
 * calls in sequence. */
tecoopsStatus_t tecoopsQkNormRotaryReshapeAndCache(
    tecoopsHandle_t handle, const int64_t *positions, long long position_stride, int axes,
    const int *sections, tecoopsRotaryLayout_t layout, void *query, void *key, const void *value,
    const void *query_weight, const void *key_weight, float eps, const int64_t *slot_mapping,
    void *key_cache, void *value_cache, int num_tokens, int num_heads, int num_kv_heads,
    int head_size, int rot_dim, long long query_stride, long long key_stride,
    long long value_stride, const float *cos_sin_cache, int max_position, float base, int is_neox,
    int num_blocks, int block_size, int write_key, tecoopsDataType_t dataType);

/* reshape_and_cache into a cache held in 4 bits.  key / value [num_tokens,
 * num_kv_heads, head_size] with token strides in elements (heads of a token
 * adjacent).  A row x of a head is held as codes n of 0..15 and a pair (scale, low)
 * of dataType that stands for scale * n + low:
 *   low = min x,  scale = (max x - min x) / 15 in fp32, rounded to dataType,
 *   n = (x - low) / scale to the nearest integer, ties to even, at most 15
 *   (0 where scale is 0);
 * a row with a NaN, or whose range is not finite in fp32, is (NaN, NaN), codes 0.
 * key_cache / value_cache uint8 [num_blocks, num_kv_heads, block_size, head_size /
 * 2], element 2j in the low half of byte j; key_scales / value_scales dataType
 * [num_blocks, num_kv_heads, block_size, 2].  Slots < 0 or past the cache are not
 * stored; a slot is at most once in a call.  head_size a multiple of 8 up to 512;
 * fewer than 2^26 (token, head) rows; strides and num_kv_heads * block_size below 2^32,
 * num_kv_heads * head_size below 2^30, num_blocks * block_size below 2^31;
 * num_tokens = 0 is done without a launch. */
tecoopsStatus_t tecoopsReshapeAndCacheInt4(tecoopsHandle_t handle, const void *key,
                                           const void *value, const int64_t *slot_mapping,
                                           void *key_cache, void *value_cache, void *key_scales,
                                           void *value_scales, int num_tokens, int num_kv_heads,
                                           int head_size, long long key_stride,
                                           long long value_stride, int num_blocks, int block_size,
                                           tecoopsDataType_t dataType);

/* Attention over that cache.  Rows, lengths, masks and bounds are those of
 * tecoopsFlashAttentionEx with cu_seqlens_q (bottom-right causal, rows of no
 * sequence and rows without a key written as zeros, the bounds shape the launch
 * alone), but the softmax has no clamp at 0, so that scores of any size are
 * weighed.  q and out [total_q, num_heads, head_size] packed; block_table int32
 * [batch, blocks_per_seq], rows block_table_stride apart; head_size in {32, 64,
 * 96, 128, 160, 192}; total_q * num_heads / num_kv_heads below 2^31, batch * num_kv_heads
 * up to 2^22.  fp16, and in bf16 up to 64 (query row, head) pairs of a kv head,
 * read K and V as they are held; longer queries in bf16 widen them to fp16 first (one
 * more rounding, finer than the output's; fp16 prompts take up to twice as long).
 * Weights and values are held relative to the largest that a query row sees: rows 2^24
 * below it and further lose digits.
 * What the cache holds behind a sequence's last key is not used, whatever it is.  A key
 * or value row of NaN, or a value row whose pair is infinite, makes the rows that see it
 * NaN and no others; large rows change nothing for the query rows that do not see them.
 * workspace: tecoopsGetFlashAttentionInt4WorkspaceSize() bytes for the same sizes
 * and bounds, 16-byte aligned; with less the keys are cut into fewer splits.  NULL
 * uses the handle's scratch, and none on a stream under capture (unsplit: slower,
 * the same result up to rounding). */
tecoopsStatus_t tecoopsFlashAttentionInt4(
    tecoopsHandle_t handle, int max_seqlen_q, int max_seqlen_k, const int *cu_seqlens_q,
    const int *kv_seq_lens, const int *block_table, long long block_table_stride, int batch,
    int blocks_per_seq, const void *q, const void *key_cache, const void *value_cache,
    const void *key_scales, const void *value_scales, void *out, int total_q, int num_heads,
    int num_kv_heads, int head_size, int num_blocks, int block_size, float softmax_scale, int causal,
    void *workspace, size_t workspace_bytes, tecoopsDataType_t dataType);
tecoopsStatus_t tecoopsGetFlashAttentionInt4WorkspaceSize(int batch, int total_q, int num_heads,
                                                          int num_kv_heads, int head_size,
                                                          int max_seqlen_q, int max_seqlen_k,
                                                          size_t *bytes);

/* y[b, n] = sum_k W[n, k] x[b, k] with W[n, k] = (code - zero) * scale, fp32
 * accumulation.  weight uint8 [n, k / 2], 16-byte aligned, code 2j of a row in the
 * low half of byte j; scales and zeros dataType [n, k / group_size] (zeros NULL: 8
 * everywhere; they need not be whole); x [batch, k], y [batch, n].  group_size a
 * multiple of 32 that divides k.  For decode batches: the weights are read again
 * for every 64 rows of x; batch = 0 is done without a launch.  n up to 2^26, batch up to
 * 2^16, n * batch below 2^27 (more rows of x in slices).  Infinite and very large x are
 * taken as the formula has them (their sums again, one weight at a time: slower).
 * workspace: tecoopsGetGemvInt4WorkspaceSize() bytes for the same sizes let few rows
 * of W be split along k; with less, or NULL, there are fewer splits (slower, the
 * same result up to fp32 rounding).  Nothing is allocated. */
tecoopsStatus_t tecoopsGemvInt4(tecoopsHandle_t handle, const void *weight, const void *scales,
                                const void *zeros, const void *x, void *y, int batch, int n, int k,
                                int group_size, void *workspace, size_t workspace_bytes,
                                tecoopsDataType_t dataType);
tecoopsStatus_t tecoopsGetGemvInt4WorkspaceSize(int batch, int n, int k, size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif  /* TECOOPS_INCLUDE_TECOOPS_H_ */
