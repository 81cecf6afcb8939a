/*
 * citlali_hip.h -- C ABI of the MI355X (gfx950) decode hot path.
 *
 * This is the drop-in boundary that replaces the reference's CUDA layer
 * (include/citlali/compute/cuda/{kernels.h,tensor.h,cuda_utils.h} and
 * src/compute/cuda/{kernels.cu,tensor.cu}).  Plain pointers and sizes only.
 *
 * Conventions (same as the reference's launch_* functions, kernels.h:8-61):
 *  - fp16 values are uint16_t bit patterns, quantised weights raw GGUF
 *    super-blocks (uint8_t), fp32 values float; all pointers are device
 *    pointers unless a parameter says "host".
 *  - weights are row-major [out_features][in_features/256] super-blocks.
 *  - every call returns CITLALI_OK or an error code; the message of the last
 *    error of the calling thread is citlali_hip_last_error().  Argument
 *    checks run before anything touches the GPU.  HIP failures read
 *    "HIP error at <file>:<line> for <expr>: <message>" (the shape of the
 *    reference's CITLALI_CUDA_CHECK, cuda_utils.h:17-22).
 *  - launches are asynchronous on the library's current stream (default: the
 *    null stream, like the reference's <<<>>> launches); D2H copies and
 *    citlali_hip_synchronize() wait for it.
 *  - alignment: quantised Q4_K weights and x vectors 16-byte aligned, Q6_K
 *    weights 4-byte aligned (any hipMalloc'd buffer qualifies).
 */
#ifndef CITLALI_HIP_H
#define CITLALI_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CITLALI_OK 0
#define CITLALI_ERR_INVALID 1     /* rejected argument, nothing launched */
#define CITLALI_ERR_UNSUPPORTED 2 /* valid for the reference, not built here */
#define CITLALI_ERR_HIP 3         /* HIP runtime error */

#define CITLALI_HIP_ABI_VERSION 1

/* ---- errors and runtime ------------------------------------------------- */

/* Replaces check_cuda/CITLALI_CUDA_CHECK (cuda_utils.h:17-26): message of the
 * calling thread's last failed call ("" if none). */
const char* citlali_hip_last_error(void);
int citlali_hip_abi_version(void);

/* Selects the device for this thread (the reference always uses device 0). */
int citlali_hip_init(int device);
int citlali_hip_device_count(int* count);

/* Stream used by every launch (hipStream_t; NULL = null stream, the
 * reference's legacy default stream). */
int citlali_hip_set_stream(void* stream);
void* citlali_hip_get_stream(void);

/* Replaces QwenModel::synchronize's cudaDeviceSynchronize
 * (qwen_model.cpp:443-445): waits for the current stream and reports any
 * asynchronous kernel fault. */
int citlali_hip_synchronize(void);

/* ---- device memory: DeviceBuffer (tensor.h:10-54, tensor.cu:49-104) ------ */

int citlali_hip_malloc(void** ptr, size_t bytes);              /* tensor.cu:49-59 (bytes == 0 -> *ptr = NULL) */
int citlali_hip_free(void* ptr);                               /* tensor.cu:67-73 */
/* tensor.cu:76-78; returns once the bytes are on the device.  Copies of 8 MB
 * and more go through two pinned 8 MB staging buffers per device (allocated
 * on first use, kept until the process ends), host threads filling one while
 * the DMA engine drains the other. */
int citlali_hip_memcpy_h2d(void* dst, const void* host_src, size_t bytes);
int citlali_hip_memcpy_d2h(void* host_dst, const void* src, size_t bytes); /* tensor.cu:88-90, waits */
int citlali_hip_memcpy_d2d(void* dst, const void* src, size_t bytes);
/* cuda_zero (kernels.h:8, kernels.cu:655-657); a fill kernel, so it is safe
 * inside captured graphs. */
int citlali_hip_zero(void* ptr, size_t bytes);

/* ---- hot path: fused dequant GEMV ---------------------------------------- *
 * y[r] = sum_k W[r,k] x[k], W dequantised in fp32 (never rounded to fp16),
 * fp32 accumulation.  in_features must be a positive multiple of 256 (the
 * reference truncates silently, kernels.cu:204; this ABI rejects it) and at
 * most CITLALI_MAX_IN_FEATURES. */
#define CITLALI_MAX_IN_FEATURES 28672

/* launch_matvec_q4k (kernels.h:26, kernels.cu:772-776); y fp16 (RNE) */
int citlali_hip_matvec_q4k(const uint8_t* w, const uint16_t* x, uint16_t* y, int in_features, int out_features);
/* Q4_K with fp32 output: no reference launcher; same kernel, fp32 store
 * (the fp32-output form the reference has for Q6_K, kernels.h:30). */
int citlali_hip_matvec_q4k_to_float(const uint8_t* w, const uint16_t* x, float* y, int in_features,
                                    int out_features);
/* launch_matvec_q6k (kernels.h:28, kernels.cu:779-783); y fp16 (RNE) */
int citlali_hip_matvec_q6k(const uint8_t* w, const uint16_t* x, uint16_t* y, int in_features, int out_features);
/* launch_matvec_q6k_to_float (kernels.h:30, kernels.cu:786-796); logits */
int citlali_hip_matvec_q6k_to_float(const uint8_t* w, const uint16_t* x, float* y, int in_features,
                                    int out_features);

/* launch_embed_q6k (kernels.h:32, kernels.cu:340-378, 670-683): row
 * token_id of a Q6_K table -> fp16, the exact fp32 value rounded
 * nearest-even as the reference kernel's __float2half store does. */
int citlali_hip_embed_q6k(const uint8_t* table, int32_t token_id, uint16_t* out, int hidden);

/* ---- hot path: decode attention ------------------------------------------ *
 * launch_attention (kernels.h:38-47, kernels.cu:846-876).  Same arguments.
 * caches [max_context][kv_heads][head_dim] fp16, positions 0..position
 * inclusive.  `scores` (heads*max_context floats, as the reference sizes it,
 * qwen_model.cpp:233) is used as the split-KV workspace when large enough;
 * otherwise the library keeps its own per-device workspace (allocated on the
 * first call that needs it, kept until citlali_hip_release_workspace()).
 * It no longer receives the raw scores.  head_dim 64 or 128, heads/kv_heads
 * between 1 and 8.  Cached values are expected finite: an Inf in V is an Inf in
 * the output of its dim (unless its weight is 0 or it lies in the last chunk of
 * several), but NaN at head_dim 128 with two heads per kv head and more, whose
 * weights are split in two for the matrix cores.  The split of the positions over workgroups is planned
 * for citlali_hip_attention_plan_length(position + 1, max_context), so all
 * steps of one such length run the same launches. */
int citlali_hip_attention(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache, float* scores,
                          uint16_t* out, int position, int max_context, int heads, int kv_heads, int head_dim);

/* Attention that allocates nothing.  No counterpart in the reference: for
 * callers that cannot allocate device memory -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.  Same
 * arguments and results as citlali_hip_attention (bit for bit, same
 * launches) without `scores`: the split-KV partials go to a file-scope
 * device array of the library, CITLALI_NOALLOC_SCRATCH_BYTES per GPU, whose
 * device address citlali_hip_init resolves (or the first call on a GPU that
 * init did not select); the GPU holds it until the process ends.  A plan
 * whose partials (heads * chunks * (head_dim + 4) * 4 bytes) exceed it --
 * more than 496 chunks at 64 query heads of head_dim 128; every plan of at
 * most 32 query heads fits (at most 512 chunks) -- is rejected with
 * CITLALI_ERR_INVALID before anything launches.  Every call on a GPU shares that GPU's array,
 * which keeps the last call's partials: calls that overlap on one GPU (from
 * several streams or threads) race. */
#define CITLALI_NOALLOC_SCRATCH_BYTES (16u << 20)
int citlali_hip_attention_noalloc(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                  uint16_t* out, int position, int max_context, int heads, int kv_heads,
                                  int head_dim);

/* Many independent sequences in one launch (no reference counterpart: the
 * reference decodes one sequence; per sequence the result equals
 * launch_attention).  q/out [nseq][heads][head_dim]; sequence s uses the
 * caches at k_cache + s*seq_stride (elements); positions: device int32
 * [nseq], each < max_positions_bound (a larger one is treated as
 * max_positions_bound - 1, so no read leaves the caches); workspace of
 * citlali_hip_attention_workspace_bytes() bytes (may be NULL if that is 0). */
int citlali_hip_attention_batched(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                  long long seq_stride, const int32_t* positions, int max_positions_bound,
                                  int nseq, int heads, int kv_heads, int head_dim, void* workspace,
                                  size_t workspace_bytes, uint16_t* out);
/* The length attention is planned for at `length` = position + 1 (no
 * reference counterpart): the smallest power of two >= max(length, 256),
 * at most max_context; 0 for length <= 0 or length > max_context.  A step
 * replayed with the position in device memory (citlali_hip_attention_batched
 * with nseq 1 and this max_positions_bound) equals citlali_hip_attention at
 * every position of the bucket, bit for bit. */
int citlali_hip_attention_plan_length(int length, int max_context);
/* Workspace bytes that hold the split-KV partials of the plan for every
 * bound in [1, max_positions_bound] (no reference counterpart; the
 * reference's scores buffer is heads*max_context floats): the planned chunk
 * count is not monotone in the length, so a buffer sized for the longest
 * length alone can be too small for a shorter bucket.  0 when no length up
 * to the bound splits. */
size_t citlali_hip_attention_workspace_bytes(int max_positions_bound, int nseq, int heads, int kv_heads,
                                             int head_dim);
/* The plan citlali_hip_attention_batched makes for this bound (and
 * citlali_hip_attention for bound = its plan length): positions per
 * workgroup and chunks of the longest sequence (no reference counterpart;
 * for tests and sizing). */
int citlali_hip_attention_plan_info(int max_positions_bound, int nseq, int heads, int kv_heads, int head_dim,
                                    int* chunk, int* n_splits);
int citlali_hip_release_workspace(void);

/* citlali_hip_qk_norm_rope_store (or its _at form) followed by
 * citlali_hip_attention (or citlali_hip_attention_batched with nseq 1 and
 * max_positions_bound plan_length) in one launch, with the same results bit
 * for bit: q is the q GEMV's output (read only, not updated), k / v the
 * step's k and v; the step's k (normed, roped) and v are stored into the
 * caches at the position and attention reads them.  The position is
 * *position_at when that is not NULL (then plan_length is the bucket, and a
 * position at or beyond it writes nothing), else `position`.  workspace:
 * citlali_hip_attention_workspace_bytes(plan length) bytes.  No reference
 * counterpart (qwen_model.cpp:315-338 makes these separate launches);
 * CITLALI_ERR_UNSUPPORTED unless head_dim is 128 with 2..8 query heads per
 * kv head. */
int citlali_hip_qk_norm_rope_store_attention(const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                             const uint16_t* q_norm, const uint16_t* k_norm, int heads,
                                             int kv_heads, int head_dim, int position, const int32_t* position_at,
                                             int plan_length, int max_context, float theta, float eps,
                                             uint16_t* k_cache, uint16_t* v_cache, void* workspace,
                                             size_t workspace_bytes, uint16_t* out);

/* launch_store_kv (kernels.h:36, kernels.cu:829-843): the cache layout
 * contract, cache[position*kv_size + i] = k[i]. */
int citlali_hip_store_kv(const uint16_t* k, const uint16_t* v, uint16_t* k_cache, uint16_t* v_cache, int position,
                         int kv_size);

/* ---- load-time dequant on the device ------------------------------------- *
 * dequant_q4_k / dequant_q6_k of weight_loader.cpp:147-323 (host rule
 * rounding, bit-exact); `count` values from ceil(count/256) blocks. */
int citlali_hip_dequant_q4k_f16(const uint8_t* w, uint64_t count, uint16_t* out);
int citlali_hip_dequant_q6k_f16(const uint8_t* w, uint64_t count, uint16_t* out);

/* ---- the rest of forward_token (kernels.h:10-36) -------------------------- */
int citlali_hip_embed(const uint16_t* table, int32_t token_id, uint16_t* out, int hidden);   /* kernels.h:10 */
int citlali_hip_copy(const uint16_t* in, uint16_t* out, int n);                              /* kernels.h:12 */
int citlali_hip_add_inplace(uint16_t* target, const uint16_t* delta, int n);                 /* kernels.h:14 */
int citlali_hip_add_bias_inplace(uint16_t* target, const uint16_t* bias, int n);             /* kernels.h:16 */
int citlali_hip_rms_norm(const uint16_t* in, const uint16_t* w, uint16_t* out, int n, float eps); /* kernels.h:18 */
int citlali_hip_rms_norm_heads(const uint16_t* in, const uint16_t* w, uint16_t* out, int heads, int head_dim,
                               float eps);                                                    /* kernels.h:20 */
int citlali_hip_matvec_fp16(const uint16_t* w, const uint16_t* x, uint16_t* y, int in_features,
                            int out_features);                                                /* kernels.h:22 */
int citlali_hip_matvec_fp16_to_float(const uint16_t* w, const uint16_t* x, float* y, int in_features,
                                     int out_features);                                       /* kernels.h:24 */
int citlali_hip_swiglu(const uint16_t* gate, const uint16_t* up, uint16_t* out, int n);      /* kernels.h:34 */
int citlali_hip_rope(uint16_t* data, int heads, int head_dim, int position, float theta);    /* kernels.h:35 */

/* Greedy sampling on the device: index of the first greatest finite logit
 * (0 if none; -0.0 equals +0.0), written to device int32 *out_index.
 * Replaces the host loop of sample_greedy_from_logits (qwen_model.cpp:
 * 448-465).  Uses a per-device partials table in the library: argmax calls
 * that overlap on one device (several streams) race. */
int citlali_hip_argmax(const float* logits, int n, int32_t* out_index);

/* ---- replayable decode steps (no reference counterpart) ------------------ *
 * A decode step whose inputs live in device memory can be captured once in
 * a HIP graph and replayed per token without host synchronisation.  The
 * decode state is device int32 state[4] = {token, position, step, 0},
 * 16-byte aligned.
 * citlali_hip_argmax_advance: citlali_hip_argmax of logits, then
 *   tokens[step] = pick (when step < capacity), token = pick, position += 1,
 *   step += 1.
 * citlali_hip_embed_q6k_at / citlali_hip_embed_at: embed_q6k / embed with the
 *   token read from `token` (device); a token outside [0, vocab) gives a
 *   zero row.
 * citlali_hip_qk_norm_rope_store_at: qk_norm_rope_store with the position
 *   read from `position` (device); a position outside [0, max_positions)
 *   writes nothing to the caches. */
int citlali_hip_argmax_advance(const float* logits, int n, int32_t* state, int32_t* tokens, int capacity);
int citlali_hip_embed_q6k_at(const uint8_t* table, const int32_t* token, int vocab, uint16_t* out, int hidden);
int citlali_hip_embed_at(const uint16_t* table, const int32_t* token, int vocab, uint16_t* out, int hidden);
int citlali_hip_qk_norm_rope_store_at(uint16_t* q, const uint16_t* k, const uint16_t* v, const uint16_t* q_norm,
                                      const uint16_t* k_norm, int heads, int kv_heads, int head_dim,
                                      const int32_t* position, int max_positions, float theta, float eps,
                                      uint16_t* k_cache, uint16_t* v_cache);
/* Streams and graphs.  citlali_hip_graph_begin starts capturing the launches
 * the calling thread makes on the library stream (which must not be the null
 * stream); citlali_hip_graph_end stops the capture (also after a failed
 * launch) and returns an executable graph, replayed on the library stream by
 * citlali_hip_graph_launch.  Nothing may allocate during a capture (the
 * attention workspace must come from the caller).  A graph keeps the
 * pointers and scalars it captured. */
int citlali_hip_stream_create(void** stream);
int citlali_hip_stream_destroy(void* stream);
int citlali_hip_graph_begin(void);
int citlali_hip_graph_end(void** graph);
int citlali_hip_graph_launch(void* graph);
int citlali_hip_graph_destroy(void* graph);

/* ---- timing (bench and tests) --------------------------------------------- */
/* Reads `bytes` (16-byte multiple) of a device buffer once, as fast as the
 * memory system allows: the measured HBM read ceiling.  `sink`: 4 bytes. */
int citlali_hip_stream_read(const void* buf, size_t bytes, void* sink);
/* ---- fused forward_token steps (no reference counterpart) ---------------- *
 * Each equals the sequence of reference launches it names, bit for bit (same
 * fp16 store points and reduction order); QwenModel uses them to cut the
 * launches per layer.                                                       */
/* launch_add_inplace(x, delta) then launch_rms_norm(x, w, out) */
int citlali_hip_add_rms_norm(uint16_t* x, const uint16_t* delta, const uint16_t* w, uint16_t* out, int n, float eps);
/* launch_rms_norm_heads on q and k (skipped for a NULL weight), launch_rope
 * on q and k, launch_store_kv(k, v) -- q rewritten in place, k and v written
 * to the caches at `position`.  head_dim even and <= 128. */
int citlali_hip_qk_norm_rope_store(uint16_t* q, const uint16_t* k, const uint16_t* v, const uint16_t* q_norm,
                                   const uint16_t* k_norm, int heads, int kv_heads, int head_dim, int position,
                                   float theta, float eps, uint16_t* k_cache, uint16_t* v_cache);
/* GEMV weight types of the grouped / fused entry points below: GGUF type
 * 12 = Q4_K or 14 = Q6_K (KeepQuantized blocks; Q4_K 16-byte, Q6_K 4-byte
 * aligned), or 1 = F16 (DequantizeToFp16 rows, the weight pointer to the
 * fp16 values, 16-byte aligned; the results equal citlali_hip_matvec_fp16 /
 * _to_float bit for bit).
 *
 * LinearBackend::forward for ffn_gate and ffn_up (both of GGUF type
 * `gguf_type`) then launch_swiglu.  Returns
 * CITLALI_ERR_UNSUPPORTED, launching nothing, for in_features other than
 * 1024, 2048, 2560, 3072, 4096, 5120 or 8192 -- then use the separate
 * launches. */
int citlali_hip_matvec_gate_up_swiglu(int gguf_type, const uint8_t* w_gate, const uint8_t* w_up, const uint16_t* x,
                                      uint16_t* act, int in_features, int out_features);
/* LinearBackend::forward (linear_backend.cpp:17-61) for `count` (1..3)
 * weights that read the same input -- attn_q, attn_k and attn_v of one
 * layer (qwen_model.cpp:315-321) -- in one launch.  gguf_types[i] is 12 =
 * Q4_K, 14 = Q6_K or 1 = F16 (all or none), outputs[i] receives
 * out_features[i] fp16 values: the results of the separate
 * citlali_hip_matvec_q4k / _q6k / _fp16 calls bit for bit.  Outputs must
 * not overlap each other or x.  Returns CITLALI_ERR_UNSUPPORTED, launching
 * nothing, for in_features other than 1024, 2048, 2560, 3072, 4096, 5120,
 * 6144, 8192, 9728, 12288 or 16384, or F16 mixed with quantized types --
 * then use the separate launches. */
int citlali_hip_matvec_group(int count, const int* gguf_types, const uint8_t* const* weights, const uint16_t* x,
                             uint16_t* const* outputs, const int* out_features, int in_features);

/* GEMVs whose input is a residual add + RMSNorm (no reference counterpart):
 * the GEMV reads fp16(s * rsqrt(mean(s^2) + eps) * weight) with
 * s = fp16(x + delta) (s = x when delta is NULL); when sum_out is not NULL
 * it receives s.  The results equal citlali_hip_add_rms_norm(x, delta,
 * weight, tmp) followed by the plain GEMV on tmp, bit for bit (same
 * reduction order), without the separate launch: the reference's
 * add_inplace + rms_norm before attn_q/k/v, ffn_gate/up and the output
 * (qwen_model.cpp:306, 340-341, 372, 385).  weight, delta and sum_out
 * 16-byte aligned; sum_out must not be x or delta.  in_features 1024,
 * 2048, 2560, 3072, 4096, 5120, 6144, 8192, 9728, 12288 or 16384 (gate_up:
 * 1024, 2048, 2560, 3072, 4096, 5120 or 8192), else CITLALI_ERR_UNSUPPORTED
 * with nothing launched. */
typedef struct citlali_hip_norm {
    const uint16_t* delta;
    const uint16_t* weight;
    uint16_t* sum_out;
    float eps;
} citlali_hip_norm;
int citlali_hip_matvec_group_norm(int count, const int* gguf_types, const uint8_t* const* weights, const uint16_t* x,
                                  const citlali_hip_norm* norm, uint16_t* const* outputs, const int* out_features,
                                  int in_features);
int citlali_hip_matvec_gate_up_swiglu_norm(int gguf_type, const uint8_t* w_gate, const uint8_t* w_up,
                                           const uint16_t* x, const citlali_hip_norm* norm, uint16_t* act,
                                           int in_features, int out_features);
/* gguf_type 12 / 14 / 1; y fp16 (f32_out 0) or fp32 (f32_out 1) */
int citlali_hip_matvec_norm(int gguf_type, const uint8_t* w, const uint16_t* x, const citlali_hip_norm* norm,
                            void* y, int f32_out, int in_features, int out_features);

/* ---- paged cache of 4-bit keys and values (no reference counterpart) ------ *
 * A cache that many sequences share page by page, each with a table of the
 * pages it holds.  A page keeps page_size tokens of every kv head at 5 bits a
 * value: head_dim * 5 / 4 bytes for a token's K and V of one head, where the
 * fp16 cache takes head_dim * 4.
 *
 * 32 dims of one token share two fp16 numbers, m = fp16(min) and
 * d = fp16((max - m) * fp32(1 / 15)); a dim's code is clamp(round((y - m) / d), 0, 15)
 * (ties to even; 0 where d is not above 0: values closer together than m's
 * rounding) and stands for fp16(d * code + m).  Values saturate at +-61440
 * first; a NaN makes its 32 dims NaN.
 *
 * A slot is page * page_size + row.  One kv head's part of a page
 * (page_bytes / kv_heads, heads in order):
 *   K codes  [page_size][head_dim / 2] bytes: 4 bytes hold 8 dims, in order
 *            (low bits first) dims 0 2 4 6 1 3 5 7
 *   K params [page_size][head_dim / 32] fp16 pairs d, m
 *   V codes  [page_size / 4][head_dim / 4][4 tokens] 16-bit words of 4 dims
 *   V params [page_size / 4][head_dim / 32] fp16 d of 4 tokens, then m
 * page_size 16, 32, 64, 128 or 256; head_dim 64 or 128; kv_heads at most 4096;
 * pages 16-byte aligned; num_pages * page_size at most INT_MAX. */
typedef struct citlali_hip_kv4_cache {
    uint8_t* pages; /* [num_pages][kv_heads][page_bytes / kv_heads] */
    int num_pages;
    int page_size;
    int kv_heads;
    int head_dim;
} citlali_hip_kv4_cache;
/* Bytes of one page; 0 for a shape the cache does not have. */
size_t citlali_hip_kv4_page_bytes(int page_size, int kv_heads, int head_dim);

/* cos and sin of position * theta^(-2i / head_dim), angles in 64 bits, for
 * citlali_hip_kv4_append: table [positions][head_dim / 2][cos, sin] floats.
 * Any other table of that shape (a scaled rotation, say) serves as well.
 * positions * head_dim / 2 at most 2^31. */
int citlali_hip_rope_table(float* table, int positions, int head_dim, float theta);

/* Appends `tokens` tokens of any sequences in one launch.  Token t's query
 * heads (q + t * q_stride, [heads][head_dim]) and key heads (k + t *
 * kv_stride, [kv_heads][head_dim]) get their RMSNorm (skipped for a NULL
 * weight) and the rotation of row positions[t] of `rope` (pairs i,
 * i + head_dim / 2); the queries go to q_out + t * q_out_stride, rounded to
 * fp16 once, the keys and v + t * kv_stride to slot slots[t] of the cache.
 * Keys are normed and rotated in 64 bits, so a code is the one its definition
 * gives.  A position outside [0, rope_positions) writes nothing for its token,
 * a slot outside the cache stores nothing: rows of a padded batch carry -1.
 * Two tokens of one call must not name one slot: the slot then holds parts of
 * both.  q may be NULL with heads 0 (keys and values only); q_out may be q
 * when the strides agree.  q, k, v and q_out 16-byte aligned, strides multiples
 * of 8 (elements); q_norm, k_norm 16-byte, rope 8-byte aligned.  heads at most
 * 4096, tokens * (heads + 2 kv_heads) 2^27.  tokens 0 launches nothing. */
int citlali_hip_kv4_append(const citlali_hip_kv4_cache* cache, const uint16_t* q, const uint16_t* k,
                           const uint16_t* v, long long q_stride, long long kv_stride, const uint16_t* q_norm,
                           const uint16_t* k_norm, float eps, const float* rope, int rope_positions,
                           const int32_t* positions, const int32_t* slots, int tokens, int heads, uint16_t* q_out,
                           long long q_out_stride);
/* The values that `count` slots hold, as fp16 rows [count][kv_heads][head_dim]
 * (16-byte aligned); a slot outside the cache reads as zeros.  count * 2 *
 * kv_heads at most 2^27; count 0 launches nothing. */
int citlali_hip_kv4_read(const citlali_hip_kv4_cache* cache, const int32_t* slots, int count, uint16_t* k_out,
                         uint16_t* v_out);

/* Causal attention over the cache: softmax(q . K / sqrt(head_dim)) V for the
 * queries of nseq sequences, which are each sequence's last positions.
 *  - Queries of sequence s are rows query_start[s] .. query_start[s + 1] - 1
 *    of q (row r at q + r * q_stride, [heads][head_dim]) and out; query_start
 *    has nseq + 1 entries and does not decrease.  NULL: one query each, row s
 *    (tokens == nseq).  Rows past the last sequence's are left as they were.
 *  - context_lens[s] positions are cached, the queries' own among them: with n
 *    queries, query i sees positions 0 .. context_lens[s] - n + i.  A query
 *    that sees none, or only scores of -inf, gives zeros; a length below 0
 *    counts as 0.
 *  - position p of sequence s is row p % page_size of page page_table[s *
 *    pages_per_seq + p / page_size]; a page outside the cache counts as not
 *    there (its positions take no part).
 *  - max_query and max_context bound the queries and the positions of a
 *    sequence: the launch is planned for them.  Queries past max_query are
 *    left as they were; positions past max_context are not read.
 *    max_context is at most pages_per_seq * page_size and 65535 * 1024.
 * What a query does not see may hold anything: slots past a sequence's
 * positions, and NaN in the keys or values of the queries behind it.  Scores
 * and sums are fp32; weights go into the product with V and into their sum as
 * fp16, scaled so that the largest is between 2^10 and 2^14.  A call is planned
 * for max_query queries of every sequence: where pieces of prompts stand beside
 * sequences with a few queries each, a call for each kind is faster (512
 * queries of one sequence and one each of 32, 32/8 heads of 128: 84 us against
 * 232 in one call).  heads / kv_heads between 1 and 16, heads at most 4096,
 * nseq at most 65535, nseq * kv_heads 2^23, max_query * heads 2^25, tokens *
 * heads 2^31.  Workspace:
 * citlali_hip_kv4_attention_workspace_bytes() of the same bounds, 16-byte
 * aligned (may be NULL if that is 0); calls that overlap need one each.  q and
 * out 16-byte aligned, strides multiples of 8.  nseq 0 or tokens 0 launches
 * nothing. */
int citlali_hip_kv4_attention(const citlali_hip_kv4_cache* cache, const uint16_t* q, long long q_stride,
                              const int32_t* query_start, const int32_t* context_lens, const int32_t* page_table,
                              int pages_per_seq, int nseq, int tokens, int max_query, int max_context, int heads,
                              void* workspace, size_t workspace_bytes, uint16_t* out, long long out_stride);
size_t citlali_hip_kv4_attention_workspace_bytes(int max_context, int max_query, int nseq, int tokens, int heads,
                                                 int kv_heads, int head_dim);

/* ---- trees of drafted tokens (no reference counterpart) -------------------- *
 * Speculative decoding: a step drafts several tokens of each sequence, the model
 * runs over all of them at once, and some of them stay.  A sequence's rows are
 * query_start[s] .. query_start[s + 1] - 1 as in citlali_hip_kv4_attention, at
 * most CITLALI_MAX_TREE.  Row 0 is the token the step before ended with; a row's
 * parent is an earlier row of the sequence, by its index there, or -1 (only the
 * positions before the tree are above it).  A chain of drafts has parents -1, 0,
 * 1, ...  One step, per layer the third and fourth call:
 *   citlali_hip_draft_tree         masks and positions of the rows
 *   (embedding, projections)
 *   citlali_hip_kv4_append         the rows' K and V, in order, as the sequence's
 *                                  last slots, rotated by those positions
 *   citlali_hip_kv4_tree_attention
 *   (output projection)
 *   citlali_hip_verify_drafts      the path that stays, and the token after it
 *   citlali_hip_kv4_keep           the path's K and V moved up, in all layers   */
#define CITLALI_MAX_TREE 256

/* masks [tokens][(max_query + 63) / 64]: bit j of a row's mask (bit j % 64 of word
 * j / 64) says whether the row sees row j of its sequence, that is itself and the
 * rows above it.  positions (may be NULL) [tokens]: the row's place in the text,
 * context_lens[s] - rows + rows above it, with the sequence's rows among the
 * context_lens[s] cached positions.  A row whose parent is neither -1 nor an
 * earlier row, and every row below it, sees nothing and has position -1.  Rows
 * past max_query, and past the last sequence's, are left as they were.  masks
 * 8-byte aligned; nseq at most 65535.  nseq 0 or tokens 0 launches nothing. */
int citlali_hip_draft_tree(const int32_t* parents, const int32_t* query_start, const int32_t* context_lens, int nseq,
                           int tokens, int max_query, uint64_t* masks, int32_t* positions);

/* citlali_hip_kv4_attention, with its arguments and limits, but for what a query
 * sees: the positions before the tree, 0 .. context_lens[s] - n - 1 of a sequence
 * with n rows, and position context_lens[s] - n + j where bit j of its mask is set
 * (any masks of that layout, not only a tree's; bits past the row count are
 * ignored).  max_query is at most CITLALI_MAX_TREE.  Workspace:
 * citlali_hip_kv4_tree_attention_workspace_bytes() of the same bounds. */
int citlali_hip_kv4_tree_attention(const citlali_hip_kv4_cache* cache, const uint16_t* q, long long q_stride,
                                   const int32_t* query_start, const int32_t* context_lens, const uint64_t* masks,
                                   const int32_t* page_table, int pages_per_seq, int nseq, int tokens, int max_query,
                                   int max_context, int heads, void* workspace, size_t workspace_bytes, uint16_t* out,
                                   long long out_stride);
size_t citlali_hip_kv4_tree_attention_workspace_bytes(int max_context, int max_query, int nseq, int tokens, int heads,
                                                      int kv_heads, int head_dim);

/* Which drafted tokens stay, so that the tokens that come out are distributed as
 * if the model had drawn them one by one.  Row r's logits (element r * row_stride
 * on; gguf_type 0 = F32 or 1 = F16) are the model's after row r's token; p is
 * softmax(logits / temperatures[s]) (NULL: 1; infinite: the tokens above -inf alike),
 * or, where the temperature is not above 0 or NaN, 1 for the largest logit (the lowest
 * id of equal ones).  uniforms has a
 * random number of [0, 1) for each row.
 *  - From row 0 on, the children of the current row are tried in order.  Child c,
 *    whose token is x, becomes the current row if u_c R < p(x), where R is 1 for a
 *    row's first child; else R loses p(x), and p(x) becomes 0.
 *  - The next token is drawn from what is left of p at the row where the path
 *    ends: the first id whose running sum exceeds u_0 times the total.
 *  - With draft_logits (chains only: parents NULL), row r's are those that row
 *    r + 1's token was drawn from, at the same temperature, q their distribution.
 *    The token becomes the current row if u q(x) < p(x); else what is left is
 *    max(p - q, 0).
 *  - Where nothing is left (numbers outside [0, 1), which count as the nearest in
 *    it, NaN as 0), the next token is drawn from p as it was.
 * parents NULL: chains.  query_start NULL: one row each, whose next token is drawn
 * (then tokens may be NULL).  A token outside [0, vocab) and one whose parent is
 * not an earlier row are never accepted; a logit of -inf is a token that cannot
 * come.  A row with a NaN, +inf or nothing above -inf has no distribution: no
 * child of it is accepted, and if the path ends there the next token is -1; with
 * such draft logits a row's child is rejected and the token drawn from p.
 * Outputs: paths [nseq][max_query], the path's rows by their index in the
 * sequence, row 0 first, then -1; counts [nseq], their number (0 for a sequence
 * without rows); next_tokens [nseq] (-1 likewise); token_probs [rows], each
 * token's p under its parent row, 0 for row 0.  paths, counts and token_probs may
 * be NULL.  Probabilities and their sums are 64-bit floats.  Rows past max_query
 * take no part.  nseq at most 65535, vocab 2^30, nseq * max_query * vocab 2^40.
 * Workspace: citlali_hip_verify_drafts_workspace_bytes() (drafts: with draft
 * logits or not), 16-byte aligned; calls that overlap need one each.  nseq 0
 * launches nothing. */
int citlali_hip_verify_drafts(const void* logits, int gguf_type, long long row_stride, int vocab,
                              const void* draft_logits, long long draft_row_stride, const int32_t* tokens,
                              const int32_t* parents, const int32_t* query_start, int nseq, int rows, int max_query,
                              const float* temperatures, const float* uniforms, int32_t* paths, int32_t* counts,
                              int32_t* next_tokens, float* token_probs, void* workspace, size_t workspace_bytes);
size_t citlali_hip_verify_drafts_workspace_bytes(int nseq, int rows, int max_query, int vocab, int drafts);

/* Moves cached tokens up within their sequences, in the caches of many layers at
 * once (same shape and page tables; n_caches at most CITLALI_MAX_KEEP_CACHES):
 * position first[s] + kept[s * kept_stride + j] of sequence s goes to position
 * first[s] + j, for j below counts[s] and max_count.  kept ascends.  After
 * citlali_hip_verify_drafts, first is the length before the tree, kept and counts
 * are its paths and counts, and the sequence's new length first[s] + counts[s];
 * any other positions of a sequence may be dropped the same way.  An entry not
 * above its j, and one whose position (or the one it goes to) has no page, moves
 * nothing; a negative first moves nothing of the sequence.  Sequences that share a
 * page must not move anything to it.  nseq * kv_heads at most 2^23, max_count 2^30.
 * nseq or max_count 0 launches nothing. */
#define CITLALI_MAX_KEEP_CACHES 128
int citlali_hip_kv4_keep(const citlali_hip_kv4_cache* caches, int n_caches, const int32_t* page_table,
                         int pages_per_seq, int nseq, const int32_t* first, const int32_t* kept,
                         long long kept_stride, const int32_t* counts, int max_count);

/* ---- log probabilities (no reference counterpart) -------------------------- *
 * For each of `rows` rows of logits (row r at element r * row_stride; gguf_type
 * 0 = F32 or 1 = F16), with natural logarithms and fp32 sums:
 *  - logprobs[r] = log softmax at tokens[r], and ranks[r], the number of tokens
 *    before it (larger logit, or equal and a lower id); a token outside
 *    [0, vocab) -- a row without one -- gives 0 and -1;
 *  - entropies[r] of the row's distribution;
 *  - top_ids / top_logprobs [rows][top_k]: the top_k most likely tokens, equal
 *    logits by the lower id first.
 * A logit of -inf is a token that cannot come (it adds nothing to the entropy).
 * A row with a NaN, +inf or nothing above -inf has no distribution: its log
 * probabilities and entropy are NaN (the ids stay ordered by logit; a NaN logit
 * is never among them and before no token).  Fewer than top_k tokens to list:
 * id -1, log probability -inf.  Outputs may be NULL: logprobs and ranks (tokens
 * may then be NULL too), entropies, and top_ids with top_logprobs when top_k is
 * 0.  top_k at most CITLALI_MAX_TOP_LOGPROBS, rows 2^23, vocab 2^30.  Workspace:
 * citlali_hip_token_logprobs_workspace_bytes(), 16-byte aligned (may be NULL if
 * that is 0); calls that overlap need one each.  rows 0 launches nothing. */
#define CITLALI_MAX_TOP_LOGPROBS 64
int citlali_hip_token_logprobs(const void* logits, int gguf_type, long long row_stride, int rows, int vocab,
                               const int32_t* tokens, float* logprobs, int32_t* ranks, float* entropies, int top_k,
                               int32_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes);
size_t citlali_hip_token_logprobs_workspace_bytes(int rows, int vocab, int top_k);

/* Kernel timing (no reference counterpart; for benchmarks): while armed with
 * two events of citlali_hip_event_create, the first kernel the calling thread
 * launches records `start` when it begins and every kernel records `stop`
 * when it ends, stamped from the dispatch itself (hipExtLaunchKernel), so
 * citlali_hip_event_elapsed_ms(start, stop) is the kernels' own time.  Arm
 * before a call, disarm with (NULL, NULL) after it. */
int citlali_hip_set_kernel_timing(void* start, void* stop);
/* Per-dispatch kernel timing (no reference counterpart; for benchmarks):
 * while armed with n pairs of events (1 <= n <= CITLALI_MAX_TIMED_DISPATCHES),
 * the i-th kernel the calling thread launches, i < n, records starts[i] when
 * it begins and stops[i] when it ends, stamped from the dispatch itself, so a
 * call of several kernels gives each kernel's own time without the gaps
 * between them.  citlali_hip_dispatch_timing_count gives how many kernels
 * were launched since arming (those past n are not stamped), also after
 * disarming with (NULL, NULL, 0).  Not together with
 * citlali_hip_set_kernel_timing, nor during graph capture. */
#define CITLALI_MAX_TIMED_DISPATCHES 64
int citlali_hip_set_dispatch_timing(void* const* starts, void* const* stops, int n);
int citlali_hip_dispatch_timing_count(int* count);
int citlali_hip_event_create(void** event);
int citlali_hip_event_record(void* event);                  /* on the current stream */
int citlali_hip_event_synchronize(void* event);
int citlali_hip_event_elapsed_ms(void* start, void* stop, float* ms);
int citlali_hip_event_destroy(void* event);

#ifdef __cplusplus
}
#endif

#endif /* CITLALI_HIP_H */
