/*
 * g4hip.h -- C ABI of the MI355X (gfx950) quantized matrix-vector library.
 *
 * Drop-in boundary for gemma4.kt's tensor layer.  Reference paths are relative to
 * lib/src/main/kotlin/io/github/lbenedetto/internal/.  The Kotlin side binds these
 * symbols with java.lang.foreign (FFM); a Kotlin FloatTensor implementation
 * overrides both matmul overloads and forwards here.
 *
 * Conventions
 *  - Every function returns an int status: G4_OK (0) or a negative G4_ERR_*.
 *    g4_last_error() returns a thread-local message for the last failure.
 *  - Weights are raw GGUF blocks uploaded once (no repacking) and stay in HBM
 *    until g4_weight_free; a weight is read-only and may be shared by every
 *    context on its device.
 *  - A g4_ctx owns a HIP stream and staging buffers.  One thread uses a context
 *    at a time (the reference runs one generation thread per LlamaState); open one
 *    context per thread for concurrency.
 *  - Host-pointer entry points are synchronous: outputs are complete on return,
 *    like FloatTensor.matmul.  *_dev entry points take device pointers and are
 *    asynchronous on the context's stream (g4_ctx_set_stream can point it at a
 *    caller's stream; g4_ctx_sync waits).
 *  - Element offsets are int64 (the reference's Int offsets overflow past 2^31).
 */
#ifndef G4HIP_H
#define G4HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes and the Kotlin exception each maps to. */
#define G4_OK 0
#define G4_ERR_INVALID_ARGUMENT (-1) /* IllegalArgumentException (null pointer, bad size, bad dims) */
#define G4_ERR_UNSUPPORTED (-2)      /* UnsupportedOperationException (GGML type id), FloatTensorFactory.kt:21 */
#define G4_ERR_OUT_OF_RANGE (-3)     /* IndexOutOfBoundsException (offset/rows past the tensor) */
#define G4_ERR_NO_DEVICE (-4)        /* IllegalStateException: no HIP device */
#define G4_ERR_DEVICE (-5)           /* IllegalStateException: HIP runtime failure */
#define G4_ERR_OUT_OF_MEMORY (-6)    /* OutOfMemoryError: device allocation failed */

/* GGML type ids accepted by g4_upload (GGMLType.kt:16-56, id = ordinal). */
#define G4_TYPE_F32 0
#define G4_TYPE_F16 1
#define G4_TYPE_Q4_0 2
#define G4_TYPE_Q8_0 8
#define G4_TYPE_Q4_K 12
#define G4_TYPE_Q5_K 13
#define G4_TYPE_Q6_K 14
#define G4_TYPE_BF16 30

typedef struct g4_ctx g4_ctx;
typedef struct g4_weight g4_weight;

/* Thread-local message of the last failing call on this thread ("" if none). */
const char *g4_last_error(void);

/* Library version, (major << 16) | minor. */
int g4_version(void);

/* Number of visible HIP devices (0 and G4_OK when there is none). */
int g4_device_count(int *count);

/* GGMLType.kt:16-30 blockSize/typeSize and byteSizeFor (:58-62) for a type id.
 * Returns G4_ERR_UNSUPPORTED for ids outside the supported set. */
int g4_type_info(int ggml_type, int *block_size, int *type_size);
int g4_byte_size(int ggml_type, int64_t n_elems, int64_t *nbytes);

/* Host-only validation of a matmul geometry against a tensor of `n_elems`
 * elements of `ggml_type`: the status g4_matmul would return before launching
 * (FloatTensor.kt:18-29 rows this_offset + i*dim1 .. +dim1, i < dim0, must lie
 * inside the tensor).  Needs no device. */
int g4_check_matmul(int ggml_type, int64_t n_elems, int64_t this_offset, int32_t dim0, int32_t dim1);

/* Open / close a context on device `ordinal` (creates the context's stream). */
int g4_open(int ordinal, g4_ctx **out);
int g4_close(g4_ctx *ctx);
/* Launch subsequent *_dev work on `stream` (a hipStream_t; NULL = the context's own). */
int g4_ctx_set_stream(g4_ctx *ctx, void *stream);
int g4_ctx_sync(g4_ctx *ctx);
int g4_ctx_device(const g4_ctx *ctx, int *ordinal);
/* Scratch for HIP graph capture.  *_dev calls keep intermediates (MoE hidden
 * vectors, attention and column-split partials, a standalone norm) in a
 * per-context device buffer that grows on demand.  A graph captured over such a
 * call keeps that buffer's address, so:
 *  - g4_ctx_reserve grows the buffer to `bytes` now (call it, or run the largest
 *    shapes once eagerly, before capturing);
 *  - a call that needs more than is reserved while its stream is capturing
 *    returns G4_ERR_INVALID_ARGUMENT and records nothing (g4_matmul_batch_dev of
 *    the types other than Q4_K then records its slower kernels, which need none);
 *  - once any call on the context has been captured, an outgrown buffer is kept
 *    allocated (graphs may still replay into it) until g4_close;
 *  - graphs of one context, and calls on it that use the buffer, run one after the
 *    other, or on a context each.
 * Eager g4_matmul_batch* calls (of more than 64 tokens, and for the types other
 * than Q4_K of several tokens on rows of more than 2048 columns) use a second
 * buffer, at least 64 MB from the first such call on, that no graph refers to and
 * whose users on different streams are ordered by the library.  g4_ctx_reserve
 * also readies as much of it, up to 128 MB; g4_ctx_scratch_bytes does not count
 * it.  Where it cannot be had, and under capture, more than 64 tokens run on the
 * 16-token kernels: fp32 sums in another order, and slower on long prompts.
 * Host-pointer calls synchronise and return G4_ERR_INVALID_ARGUMENT under capture.
 * No counterpart in the reference (its matmul is synchronous CPU code). */
int g4_ctx_reserve(g4_ctx *ctx, int64_t bytes);
int g4_ctx_scratch_bytes(const g4_ctx *ctx, int64_t *bytes);

/* FloatTensorFactory.kt:7-23 create(ggmlType, entry) + the GGUF slice of
 * GGUF.kt:195-212: copy `nbytes` raw GGUF bytes holding `n_elems` elements to HBM.
 * nbytes must equal byteSizeFor(n_elems) (GGMLType.kt:58-62). */
int g4_upload(g4_ctx *ctx, int ggml_type, const void *raw, int64_t nbytes, int64_t n_elems, g4_weight **out);
int g4_weight_free(g4_weight *w);
int g4_weight_info(const g4_weight *w, int *ggml_type, int64_t *n_elems, int64_t *nbytes);
/* Device address of the uploaded blocks (read-only; for callers that launch on it). */
int g4_weight_device_ptr(const g4_weight *w, const void **dptr);

/* FloatTensor.matmul(that, out, dim0, dim1, thisOffset), FloatTensor.kt:18-29:
 *   out[i] = dot(this_offset + i*dim1, that, 0, dim1) for i in [0, dim0).
 * that: host float[dim1], out: host float[dim0].  Synchronous. */
int g4_matmul(g4_ctx *ctx, const g4_weight *w, int64_t this_offset, const float *that, float *out,
              int32_t dim0, int32_t dim1);
int g4_matmul_dev(g4_ctx *ctx, const g4_weight *w, int64_t this_offset, const float *d_that, float *d_out,
                  int32_t dim0, int32_t dim1);

/* M independent activations (rows of X, row-major [M x dim1]) against the same
 * weight: Y[m*dim0 + i] = dot(this_offset + i*dim1, X[m], 0, dim1).  The reference
 * has no batched call; this is what M calls of matmul compute (Llama.kt:435-436). */
int g4_matmul_batch(g4_ctx *ctx, const g4_weight *w, int64_t this_offset, const float *X, int32_t M, float *Y,
                    int32_t dim0, int32_t dim1);
int g4_matmul_batch_dev(g4_ctx *ctx, const g4_weight *w, int64_t this_offset, const float *d_X, int32_t M,
                        float *d_Y, int32_t dim0, int32_t dim1);

/* LM head: logits = matmul(...) (Llama.kt:402) and *index = argmax(logits)
 * (FloatTensor.kt:53-66: first index of the maximum; a NaN at index 0 wins,
 * NaN elsewhere never does).  logits may be NULL when only the index is wanted. */
int g4_matmul_argmax(g4_ctx *ctx, const g4_weight *w, int64_t this_offset, const float *that, float *logits,
                     int32_t *index, int32_t dim0, int32_t dim1);
int g4_matmul_argmax_dev(g4_ctx *ctx, const g4_weight *w, int64_t this_offset, const float *d_that,
                         float *d_logits, int32_t *d_index, int32_t dim0, int32_t dim1);

/* FloatTensor.argmax(offset=0, size=n) of a float vector (FloatTensor.kt:53-66). */
int g4_argmax(g4_ctx *ctx, const float *v, int32_t n, int32_t *index);
int g4_argmax_dev(g4_ctx *ctx, const float *d_v, int32_t n, int32_t *d_index);

/* Per-element get() of every format (Q8_0FloatTensor.kt:21-28, Q4_0FloatTensor.kt:21-39,
 * Q4_KFloatTensor.kt:23-55, F16FloatTensor.kt:20-23, BF16FloatTensor.kt:20-24,
 * F32FloatTensor.kt:18-20): out[i] = get(offset + i), bit-exact; the embedding
 * lookup copyTo of Llama.kt:112. */
int g4_dequant(g4_ctx *ctx, const g4_weight *w, int64_t offset, int64_t n, float *out);
int g4_dequant_dev(g4_ctx *ctx, const g4_weight *w, int64_t offset, int64_t n, float *d_out);

/* FFN of one token (Llama.kt:357-361, MoE shared MLP :232-236):
 *   h = gelu(w_gate x) * (w_up x)  (gelu of Llama.kt:23-25),  y = w_down h.
 * w_gate, w_up: [hidden x dim], w_down: [dim x hidden]; x: float[dim], y: float[dim]. */
int g4_ffn(g4_ctx *ctx, const g4_weight *w_gate, const g4_weight *w_up, const g4_weight *w_down, const float *x,
           float *y, int32_t dim, int32_t hidden);
int g4_ffn_dev(g4_ctx *ctx, const g4_weight *w_gate, const g4_weight *w_up, const g4_weight *w_down,
               const float *d_x, float *d_y, int32_t dim, int32_t hidden);
/* The first half of that FFN (Llama.kt:357-360): h = gelu(w_gate x) * (w_up x),
 * h: float[hidden].  One fused launch; g4_ffn is this plus g4_matmul of w_down. */
int g4_ffn_gate_up(g4_ctx *ctx, const g4_weight *w_gate, const g4_weight *w_up, const float *x, float *h,
                   int32_t dim, int32_t hidden);
int g4_ffn_gate_up_dev(g4_ctx *ctx, const g4_weight *w_gate, const g4_weight *w_up, const float *d_x, float *d_h,
                       int32_t dim, int32_t hidden);

/* MoE routing of T tokens (Llama.kt:269-293): per token softmax over n_experts
 * router logits (MutableFloatTensor.kt:54-59, exp in double), top-k by repeated
 * strict-> scans (ties to the lowest index).  weights[t*k+j] = p (renormalize = 0,
 * the reference) or p / sum of the k chosen p in fp32, j order (renormalize = 1);
 * then times expert_scale[e] when expert_scale != NULL (ffn_down_exps_scale,
 * Llama.kt:302,334).  logits [T x n_experts]; ids, weights [T x k]. */
int g4_moe_route(g4_ctx *ctx, const float *logits, int32_t T, int32_t n_experts, int32_t k, int32_t renormalize,
                 const float *expert_scale, int32_t *ids, float *weights);
int g4_moe_route_dev(g4_ctx *ctx, const float *d_logits, int32_t T, int32_t n_experts, int32_t k,
                     int32_t renormalize, const float *d_expert_scale, int32_t *d_ids, float *d_weights);

/* Routed expert FFN (Llama.kt:300-337) for T tokens:
 *   Y[t] = sum_j weights[t,j] * down_e( gelu(gate_e X[t]) * up_e X[t] ),  e = ids[t,j]
 * w_gate_up: [n_experts x 2*ff x dim] (gate rows first, then up rows, per expert,
 * slab offset e*2*ff*dim); w_down: [n_experts x dim x ff] (offset e*dim*ff).
 * X [T x dim], ids/weights [T x k], Y [T x dim].
 * g4_moe checks every id against the experts the weights hold
 * (G4_ERR_OUT_OF_RANGE).  g4_moe_dev cannot (the ids are device memory): a slot
 * whose id lies outside [0, n_experts) contributes nothing (its hidden vector
 * and down rows are zero), so Y is the weighted sum over the valid slots.
 * Calls of 41 or more tokens with Q4_K weights (dim and ff multiples of 128 up
 * to 3072, at most 4096 (token, slot) pairs) run the experts grouped by expert
 * on the matrix cores: every dot within the same bound, but rounded differently
 * from the same tokens in smaller calls. */
int g4_moe(g4_ctx *ctx, const g4_weight *w_gate_up, const g4_weight *w_down, const float *X, int32_t T,
           int32_t dim, int32_t ff, const int32_t *ids, const float *weights, int32_t k, float *Y);
int g4_moe_dev(g4_ctx *ctx, const g4_weight *w_gate_up, const g4_weight *w_down, const float *d_X, int32_t T,
               int32_t dim, int32_t ff, const int32_t *d_ids, const float *d_weights, int32_t k, float *d_Y);

/* The routed MoE block of Llama.kt:269-337 from the router logits, in one call:
 * the routing of g4_moe_route (softmax, top-k, renormalize, expert_scale) and the
 * expert FFN and weighted sum of g4_moe.  logits [T x n_experts] (n_experts at
 * most the experts the weights hold); the routing is also returned in ids and
 * weights [T x k].  Up to 256 experts the routing runs inside the gate+up launch
 * (each workgroup routes its own token); above that, and for the calls that run
 * the experts grouped (see g4_moe), in a launch of its own.
 * Results are identical to g4_moe_route followed by g4_moe. */
int g4_moe_routed(g4_ctx *ctx, const g4_weight *w_gate_up, const g4_weight *w_down, const float *X, int32_t T,
                  int32_t dim, int32_t ff, const float *logits, int32_t n_experts, int32_t k, int32_t renormalize,
                  const float *expert_scale, int32_t *ids, float *weights, float *Y);
int g4_moe_routed_dev(g4_ctx *ctx, const g4_weight *w_gate_up, const g4_weight *w_down, const float *d_X, int32_t T,
                      int32_t dim, int32_t ff, const float *d_logits, int32_t n_experts, int32_t k,
                      int32_t renormalize, const float *d_expert_scale, int32_t *d_ids, float *d_weights,
                      float *d_Y);

/* g4_moe_routed_dev without any device allocation, for callers that cannot
 * allocate (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).  No counterpart in the reference.  Same arguments, results
 * and bits as g4_moe_routed_dev; its intermediates live in a fixed 16 MiB device
 * array per GPU (held until the process ends) instead of the context's scratch,
 * so 4 * T * k * (3 * ff + dim) bytes (each part rounded up to 256) must fit:
 * larger calls return G4_ERR_INVALID_ARGUMENT.  Every call on one GPU shares
 * that array: calls that overlap on one GPU (other threads, other streams or
 * contexts) race and must be serialised by the caller. */
int g4_moe_routed_dev_noalloc(g4_ctx *ctx, const g4_weight *w_gate_up, const g4_weight *w_down, const float *d_X,
                              int32_t T, int32_t dim, int32_t ff, const float *d_logits, int32_t n_experts, int32_t k,
                              int32_t renormalize, const float *d_expert_scale, int32_t *d_ids, float *d_weights,
                              float *d_Y);

/* ---- Decode step around the matvec: the activations stay in device memory. ----
 * Norm weights are uploaded F32 tensors (ModelLoader.kt:281-286 reads norms as
 * FloatBuffers and throws UnsupportedOperationException for any other type).
 * s = (float)(1.0 / sqrt((double)(ss / size + eps))), ss = fp32 sum of x*x. */
#define G4_NORM_WEIGHT_AFTER 0 /* Llama.kt:27-37 rmsnorm(out, x, weight, size, eps): w * (s * x) */
#define G4_NORM_WEIGHT_FIRST 1 /* Llama.kt:39-60 rmsnorm(out, outOffset, x, xOffset, ...): w * s * x */
#define G4_NORM_NO_WEIGHT 2    /* Llama.kt:62-78 rmsnormNoWeight: s * x */

/* rms norm of n_vec vectors of `size` floats (vector v at d_x + v*size; the per-head
 * q/k/v norms of Llama.kt:161-163, 185-188), each with its own scale and the shared
 * weight (NULL for G4_NORM_NO_WEIGHT).  d_out may be d_x (in place). */
int g4_rmsnorm_dev(g4_ctx *ctx, const g4_weight *weight, const float *d_x, float *d_out, int32_t n_vec, int32_t size,
                   float eps, int form);
/* Post-norm plus residual (Llama.kt:222-223, 362-363): v = rmsnorm(v) (the
 * G4_NORM_WEIGHT_AFTER form, in place), then x += v.  One launch. */
int g4_rmsnorm_add_dev(g4_ctx *ctx, const g4_weight *weight, float *d_v, float *d_x, int32_t size, float eps);
/* MutableFloatTensor.kt:28-37 addInPlace: x[i] = x[i] + that[i]. */
int g4_add_dev(g4_ctx *ctx, float *d_x, const float *d_that, int32_t n);
/* Llama.kt:403-406 final logit soft-capping in place: v = cap * (float)tanh((double)(v / cap)), cap > 0. */
int g4_softcap_dev(g4_ctx *ctx, float *d_v, int32_t n, float cap);
/* Norm then matmul (Llama.kt:155-158: xb = rmsnorm(x, weight); W.matmul(xb, out, dim0, dim1)):
 * out = W . rmsnorm(x) with the G4_NORM_WEIGHT_AFTER form fused into the matvec's
 * staging of x.  d_xnorm (NULL, or not overlapping d_x) receives rmsnorm(x). */
int g4_matmul_norm_dev(g4_ctx *ctx, const g4_weight *w, int64_t this_offset, const g4_weight *norm, const float *d_x,
                       float eps, float *d_xnorm, float *d_out, int32_t dim0, int32_t dim1);
/* Dense FFN block of one token, in place on x (Llama.kt:355-363):
 *   xb = rmsnorm(x, norm_pre); h = gelu(w_gate xb) * (w_up xb); xb = rmsnorm(w_down h, norm_post); x += xb.
 * Three launches: gate/up with the fused pre-norm, down, post-norm plus residual. */
int g4_ffn_block(g4_ctx *ctx, const g4_weight *w_gate, const g4_weight *w_up, const g4_weight *w_down,
                 const g4_weight *norm_pre, const g4_weight *norm_post, float *x, int32_t dim, int32_t hidden,
                 float eps);
int g4_ffn_block_dev(g4_ctx *ctx, const g4_weight *w_gate, const g4_weight *w_up, const g4_weight *w_down,
                     const g4_weight *norm_pre, const g4_weight *norm_post, float *d_x, int32_t dim, int32_t hidden,
                     float eps);
/* Final norm, logits and greedy pick (Llama.kt:401-407, then Sampler.ARGMAX =
 * FloatTensor.argmax, FloatTensor.kt:53-66):
 *   logits = W_cls . rmsnorm(x, norm_final); if softcap > 0: logits = softcap(logits); index = argmax(logits).
 * logits may be NULL; d_xnorm (device form, NULL or not overlapping d_x) receives
 * rmsnorm(x), which the reference leaves in x. */
int g4_lm_head(g4_ctx *ctx, const g4_weight *w_cls, const g4_weight *norm_final, const float *x, float *logits,
               int32_t *index, int32_t vocab, int32_t dim, float eps, float softcap);
int g4_lm_head_dev(g4_ctx *ctx, const g4_weight *w_cls, const g4_weight *norm_final, const float *d_x, float *d_xnorm,
                   float *d_logits, int32_t *d_index, int32_t vocab, int32_t dim, float eps, float softcap);

/* Decode attention of one token over one layer's KV cache (Llama.kt:198-218):
 *   for each query head h (kv head h / (n_heads / n_kv_heads)), scores
 *   s_t = q_h . K[t] with scale 1 for t = att_start..position, softmax
 *   (MutableFloatTensor.kt:54-59: max, exp in double), out_h = sum_t a_t V[t].
 * d_q, d_out: [n_heads x head_size]; d_key_cache, d_value_cache: fp32 rows of
 * kv_dim = n_kv_heads * head_size floats, row t at t * kv_dim, holding at least
 * position + 1 rows.  att_start = max(0, position - window + 1) on sliding-window
 * layers, 0 otherwise (Llama.kt:197).  Head sizes 64/128/256/512 with 16-byte
 * aligned buffers take the split-sequence kernel (two launches); any other shape
 * takes a one-workgroup-per-head kernel. */
int g4_attention_dev(g4_ctx *ctx, const float *d_q, const float *d_key_cache, const float *d_value_cache,
                     float *d_out, int32_t n_heads, int32_t n_kv_heads, int32_t head_size, int32_t position,
                     int32_t att_start);

/* ---- Paged key-value cache of several sequences, and the operators on it. ----
 * The reference keeps one sequence's keys and values in contiguous fp32 rows
 * (Llama.kt:190-218); a program that serves several shares pages between them.
 * The caller owns the memory (all of it device memory of the context's device):
 *   k, v     [n_layers][n_pages][n_kv_heads][page_tokens][head_size] of `type`
 *            (F32, F16 or BF16), 16-byte aligned
 *   table    int32 [max_seqs][max_pages]: the page of tokens j * page_tokens .. of
 *            a sequence, -1 where there is none
 *   lengths  int32 [max_seqs]: tokens of each sequence (0: none)
 *   refs     int32 [n_pages]: sequences that hold a page (0: free)
 *   status   int32 [1]
 * head_size is a multiple of 8 up to 512, page_tokens a power of two from 16 to 256,
 * max_seqs at most 1024, n_pages * page_tokens below 2^31 and max_pages *
 * page_tokens at most 2^30.  Full pages may be shared; a partly filled one has one
 * owner (the calls below keep it so).
 *
 * The calls take lists of sequences, and lengths change, in device memory: a
 * captured step advances when it is replayed.  A list names no more than 1024
 * sequences.  What a call finds there cannot be returned by it: a call that cannot
 * be done leaves the cache as it was and sets *status (1: not enough free pages, 2: an
 * index, count or length out of range, or a sequence twice), and while that is set
 * every call on the cache, attention too, does nothing.  g4_kv_status reads and
 * clears it.  Pages and lengths out of range are never followed: attention takes
 * such a page's tokens as not there.
 * Calls on one cache from several streams are the caller's to order. */
typedef struct g4_kv {
  int32_t type;
  int32_t n_layers;
  int32_t n_kv_heads;
  int32_t head_size;
  int32_t page_tokens;
  int32_t n_pages;
  int32_t max_seqs;
  int32_t max_pages;
  void *k;
  void *v;
  int32_t *table;
  int32_t *lengths;
  int32_t *refs;
  int32_t *status;
} g4_kv;

/* Host-only validation of a cache's description: the status the calls would return
 * (G4_ERR_UNSUPPORTED for another type).  Needs no device. */
int g4_kv_check(const g4_kv *kv);
/* An empty cache: every page free, no sequence. */
int g4_kv_init_dev(g4_ctx *ctx, const g4_kv *kv);
/* Waits for the context's stream and returns what *status held, which is cleared: G4_OK,
 * G4_ERR_OUT_OF_MEMORY (1) or G4_ERR_OUT_OF_RANGE (2).  Not under capture. */
int g4_kv_status(g4_ctx *ctx, const g4_kv *kv);
/* Sequence d_seqs[i] grows by d_counts[i] >= 0 tokens, whose rows are then to be
 * written (g4_kv_rope_write_dev, layer by layer).  Fresh pages are the lowest free
 * ones, in the order of the list.  One launch. */
int g4_kv_extend_dev(g4_ctx *ctx, const g4_kv *kv, int32_t n, const int32_t *d_seqs, const int32_t *d_counts);
/* Sequence d_dst[i] becomes the first d_lengths[i] tokens of d_src[i] (d_lengths NULL:
 * all of them): whole pages are shared, a partly used last page is copied to a fresh
 * one, in all layers, and what d_dst[i] held is given back.  A sequence may be the
 * source of several and itself be replaced (beams that are reordered): all read the
 * state before the call.  d_src[i] = d_dst[i] shortens, and copies nothing where the last
 * page is its own and no other entry shares it.  Fresh pages are free before the call.
 * Two launches. */
int g4_kv_fork_dev(g4_ctx *ctx, const g4_kv *kv, int32_t n, const int32_t *d_src, const int32_t *d_dst,
                   const int32_t *d_lengths);
/* Sequence d_dst[i] becomes the first d_prefix[i] tokens of d_src[i] (d_prefix NULL: none),
 * shared and copied as by g4_kv_fork_dev, followed by its tokens d_keep[j] for j in
 * [d_keep_begin[i], d_keep_begin[i + 1]), copied to fresh pages.  d_keep_begin has n + 1
 * rising entries from 0 to at most n_keep.  Keys keep the positions they were rotated
 * to.  Three launches. */
int g4_kv_compact_dev(g4_ctx *ctx, const g4_kv *kv, int32_t n, const int32_t *d_src, const int32_t *d_dst,
                      const int32_t *d_prefix, const int32_t *d_keep, const int32_t *d_keep_begin, int32_t n_keep);
/* The sequences' pages are given back; their length is 0. */
int g4_kv_free_dev(g4_ctx *ctx, const g4_kv *kv, int32_t n, const int32_t *d_seqs);
/* The pages are given back that no later token sees under a window and `sinks` first
 * tokens (see g4_paged_attention_dev).  Lengths stay.  For sequences whose last rows
 * have been attended to, before they are extended. */
int g4_kv_trim_dev(g4_ctx *ctx, const g4_kv *kv, int32_t n, const int32_t *d_seqs, int32_t window, int32_t sinks);

/* Rotary positions.  Pair i < rot / 2 of a head's first `rot` elements is turned by
 * the angle position * freqs[i], and multiplied by gain; the other elements stay.
 * G4_ROPE_HALF: pair i is elements i and i + rot / 2; G4_ROPE_PAIRS: 2i and 2i + 1.
 * Angles are formed in double precision.  (RotaryPositionEmbeddings.kt:7-54 are the
 * reference's tables.) */
#define G4_ROPE_HALF 0
#define G4_ROPE_PAIRS 1
typedef struct g4_rope {
  const double *freqs; /* device memory, rot / 2 entries */
  int32_t rot;         /* even, at most head_size */
  int32_t layout;
  float gain;
} g4_rope;

/* How positions beyond the trained length are scaled, by `factor` >= 1:
 * NONE    freqs[i] = base^(-2i / rot)
 * LINEAR  those / factor
 * BASE    with base * factor^(rot / (rot - 2)) (rot > 2)
 * RAMP    pairs that turn more than `fast` times over the `trained` length keep their
 *         frequency, those that turn less than `slow` times are divided by factor, with
 *         a linear ramp over i between; gain = 1 + ln(factor) / 10 */
#define G4_ROPE_SCALE_NONE 0
#define G4_ROPE_SCALE_LINEAR 1
#define G4_ROPE_SCALE_BASE 2
#define G4_ROPE_SCALE_RAMP 3
/* Host only: the frequencies and gain of g4_rope.  divisors (NULL, or rot / 2 positive
 * floats) divide the unscaled frequencies. */
int g4_rope_freqs(int32_t rot, double base, int32_t scaling, double factor, double trained, double fast, double slow,
                  const float *divisors, double *freqs, float *gain);
/* d_out[r] = the heads of d_x[r] turned to d_positions[r]: [n_rows][n_heads][head_size],
 * head_size even.  d_out may be d_x.  One launch. */
int g4_rope_dev(g4_ctx *ctx, const g4_rope *rope, const float *d_x, float *d_out, int32_t n_rows, int32_t n_heads,
                int32_t head_size, const int32_t *d_positions);
/* The new rows of a layer: sequence d_seqs[i] owns rows d_row_begin[i] ..
 * d_row_begin[i + 1] - 1 of n_rows (d_row_begin, n + 1 rising entries; NULL: row i), which
 * are its last tokens, so that row j stands at position length - rows + j.
 * d_q [n_rows][n_heads][head_size] is turned to d_q_out (which may be d_q; both NULL: no
 * queries), d_k [n_rows][n_kv_heads][head_size] is turned and d_v taken as it is, and
 * both are written to the sequence's pages, rounded to nearest (F16 overflows to
 * infinity).  rope NULL: nothing is turned, and d_q is NULL.  Rows of no sequence
 * are left as they are.  All or nothing: if a row's page is not there or is shared, a sequence
 * with rows is named twice, or d_row_begin does not rise, nothing is written, to d_q_out
 * neither, and *status is set.  One launch, two for more than 2048 rows. */
int g4_kv_rope_write_dev(g4_ctx *ctx, const g4_kv *kv, int32_t layer, const g4_rope *rope, const float *d_q,
                         float *d_q_out, const float *d_k, const float *d_v, int32_t n_heads, int32_t n,
                         const int32_t *d_seqs, const int32_t *d_row_begin, int32_t n_rows);

/* Decode attention over the cache (Llama.kt:198-218 for every sequence of a list): row
 * i of d_q and d_out [n][n_heads][head_size] is the last token of sequence d_seqs[i], at
 * position p = length - 1.  Head h reads kv head h / (n_heads / n_kv_heads).  With
 * scores s_t = scale * q . K[t],
 *   out = sum_t exp(s_t - max) V[t] / sum_t exp(s_t - max)
 * over the tokens t <= p that it sees: all (window = 0), or t > p - window and the
 * first `sinks`.  A row that sees nothing (an empty sequence, pages given back, scores
 * that are all -infinity) is zeros.  fp32 products and sums; over an F16 cache an element
 * of a query is taken to 2^-39 of the largest of its head.  d_q and d_out are 16-byte
 * aligned and do not overlap.  Two launches. */
int g4_paged_attention_dev(g4_ctx *ctx, const g4_kv *kv, int32_t layer, const float *d_q, float *d_out,
                           int32_t n_heads, int32_t n, const int32_t *d_seqs, float scale, int32_t window,
                           int32_t sinks);
/* The same for several tokens per sequence (prompts, their chunks, drafted tokens): the
 * rows of each sequence as in g4_kv_rope_write_dev, each at its own position and seeing
 * no later one.  Over an F16 cache queries and weights are taken to 22 bits (2^-22 of each,
 * and 2^-39 of the largest element of a query's head).  Rows of no sequence are left as they
 * are; if d_row_begin does not rise, all are, and *status is set.  Three launches. */
int g4_paged_prompt_dev(g4_ctx *ctx, const g4_kv *kv, int32_t layer, const float *d_q, float *d_out, int32_t n_heads,
                        int32_t n, const int32_t *d_seqs, const int32_t *d_row_begin, int32_t n_rows, float scale,
                        int32_t window, int32_t sinks);

#ifdef __cplusplus
}
#endif
#endif
