/*
 * intllm_hip.h — C ABI of libintllm_hip: the Q16.48 (int64 fixed-point)
 * Llama forward pass of nmicic/int-llm's llama_int, on one AMD MI355X.
 *
 * The reference has no FFI for this path: its hot path is `static` C
 * functions in llama_int.c.  Each entry point below replaces one of them
 * (cited as reference file:line) with the same argument meaning and the
 * same bits: every output equals the reference's CPU result exactly.
 *
 * Conventions
 *   - Every int64_t* / int* argument of an op is a DEVICE pointer owned
 *     by the caller (allocate with q48_malloc or any HIP allocator).
 *     Arguments off the boundary of their type are refused (Q48_EINVAL) by the
 *     ops that could fault on them.
 *   - Values are Q16.48 fixed point (`fixed_t`, fp_math.h:175).
 *   - Ops are enqueued on the context's stream, in call order; q48_sync
 *     waits for them.  Results are visible after q48_sync or a
 *     q48_memcpy_d2h (which is synchronous).
 *   - Return 0 (Q48_OK) or a negative Q48_E* code; nothing aborts.
 *     q48_strerror turns a code into text.
 *   - One context per host thread.  The reference is single-threaded
 *     (llama_int.c has no threads); contexts are independent.
 */
#ifndef INTLLM_HIP_H
#define INTLLM_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define Q48_OK          0
#define Q48_EINVAL     (-1)   /* bad argument (null pointer, size <= 0, shape) */
#define Q48_ENOMEM     (-2)   /* device allocation failed                     */
#define Q48_EHIP       (-3)   /* HIP runtime / launch error                    */
#define Q48_ERANGE     (-4)   /* token or position out of range               */
#define Q48_ESTATE     (-5)   /* op needs state not yet set up (rope tables)  */
#define Q48_ETIMEOUT   (-6)   /* a one-launch split attention could not finish */
#define Q48_ETOOBIG    (-7)   /* size exceeds the allocation-free scratch      */

typedef struct q48_ctx q48_ctx;

/* ---- context, memory, stream -------------------------------------------- */

/* Create a context on HIP device `device`: a stream of default priority and
 * the fp_math constants (FP_PI, CORDIC angles and gain) computed on the
 * device exactly as fp_math_init does (fp_math.h:833-858). */
int q48_ctx_create(q48_ctx **out, int device);
/* The same with ops enqueued on the caller's stream (a hipStream_t of that
 * device, NULL for the default stream) instead of one of the context's own,
 * so that they are ordered with what the caller enqueues there: a context's
 * own stream is ordered with no other, the default stream included, and only
 * synchronising both sides makes data pass.  The stream outlives the context.
 * Capture it with q48_graph_* (not the default stream: Q48_ESTATE, from the
 * host's q48h_decode_graph too).  While the caller captures it by other means,
 * ops that use a workspace or the one-launch split attention return
 * Q48_ESTATE, and so does this call. */
int q48_ctx_create_on(q48_ctx **out, int device, void *stream);
int q48_ctx_destroy(q48_ctx *ctx);

int q48_malloc(q48_ctx *ctx, void **dptr, size_t bytes);
int q48_free(q48_ctx *ctx, void *dptr);
/* Synchronous copies (the stream is drained first). */
int q48_memcpy_h2d(q48_ctx *ctx, void *dst, const void *src, size_t bytes);
int q48_memcpy_d2h(q48_ctx *ctx, void *dst, const void *src, size_t bytes);
/* Stream-ordered device-to-device copy. */
int q48_memcpy_d2d(q48_ctx *ctx, void *dst, const void *src, size_t bytes);
/* Stream-ordered zero fill (a kernel, so it may be graph-captured).
 * Replaces kv_cache_reset's memset (llama_int.c:1170-1183). */
int q48_zero(q48_ctx *ctx, void *dptr, size_t bytes);
int q48_sync(q48_ctx *ctx);
const char *q48_strerror(int code);

/* ---- the six hot-path ops ------------------------------------------------ */

/* y[i] = (int64)((sum_j (int128)W[i*K + j] * x[j]) >> 48), i < M.
 * Replaces matmul_vec(out, weight, in, M, N=K)  (llama_int.c:1014-1046). */
int q48_gemv(q48_ctx *ctx, int64_t *y, const int64_t *W, const int64_t *x,
             int M, int K);

/* Batched prefill: Y[t][i] = matmul_vec row i of token t, for t < T.
 * W [N][K], X [T][K], Y [T][N].  Each element is exactly what
 * matmul_vec gives for that token (llama_int.c:1014-1046 per token; the
 * reference prefills one token at a time, llama_int.c:3081-3092). */
int q48_gemm(q48_ctx *ctx, int64_t *Y, const int64_t *W, const int64_t *X,
             int T, int N, int K);

/* q48_gemm with the kernel named: Q48_GEMM_VALU multiplies 32-bit limbs on
 * the vector ALUs; Q48_GEMM_I8 splits both operands into int8 digits and
 * multiplies them on the matrix cores (v_mfma_i32_32x32x32_i8), with the
 * split either inside the k loop (Q48_GEMM_I8_FUSED) or done once per call
 * into digit planes that the k loop reads by DMA (Q48_GEMM_I8_PLANES);
 * Q48_GEMM_I8 picks one of the two by shape, and Q48_GEMM_AUTO is q48_gemm's
 * choice (the decode GEMV for T = 1, else Q48_GEMM_I8).  All give the same
 * bits.  No reference counterpart: it exists so that callers and benchmarks
 * can compare the kernels on the same inputs. */
#define Q48_GEMM_AUTO      0
#define Q48_GEMM_VALU      1
#define Q48_GEMM_I8        2
#define Q48_GEMM_I8_FUSED  3
#define Q48_GEMM_I8_PLANES 4
int q48_gemm_ex(q48_ctx *ctx, int64_t *Y, const int64_t *W, const int64_t *X,
                int T, int N, int K, int kernel);

/* A weight matrix's digit planes, prepared once for every later q48_gemm on
 * it (the int8 kernel otherwise splits W into planes in each call that
 * takes the planes path).  q48_gemm_planes_bytes gives the size of the
 * buffer (device memory the caller owns, 16-byte aligned; about 8 bytes per
 * weight); q48_gemm_prepare fills it from W [N][K]; q48_gemm_prepared is
 * q48_gemm over W with those planes (W itself is still read where a block's
 * digits leave the int8 kernel's window, and for T = 1).  Same bits as
 * q48_gemm.  The planes describe W as it was when prepared: prepare again
 * after W changes.  No reference counterpart (the reference has no batched
 * prefill): it exists for callers that run many prefills over one model. */
int q48_gemm_planes_bytes(int N, int K, size_t *bytes);
int q48_gemm_prepare(q48_ctx *ctx, void *Wp, const int64_t *W, int N, int K);
int q48_gemm_prepared(q48_ctx *ctx, int64_t *Y, const int64_t *W, const void *Wp,
                      const int64_t *X, int T, int N, int K);

/* out = rmsnorm(x) * w.  Replaces rmsnorm (llama_int.c:1048-1058). */
int q48_rmsnorm(q48_ctx *ctx, int64_t *out, const int64_t *x,
                const int64_t *w, int dim);

/* Build the RoPE cos/sin tables [max_seq][head_dim/2] on the device.
 * Replaces rope_init (llama_int.c:960-986); same bits. */
int q48_rope_init(q48_ctx *ctx, int head_dim, int max_seq, int theta);

/* Rotate n_heads consecutive head vectors of vec in place at `pos`.
 * Replaces the rope_apply loops (llama_int.c:997-1008, 1392-1395). */
int q48_rope(q48_ctx *ctx, int64_t *vec, int n_heads, int head_dim, int pos);

/* Store k_new / v_new ([n_kv][head_dim]) at cache[layer][pos] and compute
 * exact GQA attention for all n_heads query heads over positions 0..pos.
 * Cache layout [layers][max_seq][n_kv][head_dim] (kv_key_at,
 * llama_int.c:1185-1195).  Replaces the KV store, scale, exact attention
 * and softmax of transformer_layer_forward (llama_int.c:1414-1416, 1433,
 * 1502-1529, 1060-1072).  q and k_new must already be rotated. */
int q48_attn_decode(q48_ctx *ctx, int64_t *out, const int64_t *q,
                    int64_t *kcache, int64_t *vcache, const int64_t *k_new,
                    const int64_t *v_new, int layer, int pos, int n_heads,
                    int n_kv, int head_dim, int max_seq);

/* out[i] = fp_mul(fp_silu(gate[i]), up[i]).  Replaces the SwiGLU loops
 * (llama_int.c:1549-1552, fp_math.h:911-921). */
int q48_silu_mul(q48_ctx *ctx, int64_t *out, const int64_t *gate,
                 const int64_t *up, int n);

/* ---- small ops of llama_forward ----------------------------------------- */

/* acc[i] += d[i] (int64, wrapping): the residual adds (llama_int.c:1535,
 * 1556). */
int q48_add(q48_ctx *ctx, int64_t *acc, const int64_t *d, int n);

/* out = table[token] ([dim] row): the embedding lookup
 * (llama_int.c:2822-2824).  The caller range-checks token as
 * llama_forward does (llama_int.c:2813-2820). */
int q48_embed(q48_ctx *ctx, int64_t *out, const int64_t *table, int token,
              int dim);

/* Greedy token: index of the first maximum of v[0..n) (argmax,
 * llama_int.c:2888-2893).  Writes *host_out; synchronises. */
int q48_argmax(q48_ctx *ctx, const int64_t *v, int n, int *host_out);

/* ---- introspection / parity hooks ---------------------------------------- */

/* Device pointers of the current RoPE tables (after q48_rope_init). */
int q48_rope_tables(q48_ctx *ctx, const int64_t **cos_t, const int64_t **sin_t);

/* Evaluate one fp_math function element-wise on the device (no reference
 * FFI counterpart: this is fp_determinism.c's evaluation step,
 * fp_determinism.c:175-195, exposed so the gate can run on the GPU).
 * func: 0 mul(x,y) 1 div(x,y) [0 where y==0] 2 sqrt 3 sqrt_fast
 * 4 inv_sqrt 5 exp 6 log 7 sincos (out0=cos, out1=sin) 8 sigmoid 9 silu
 * 10 safe_exp 11 exp_dyadic(x, k=y) 12 div(x,y) [0 where y==0] through the
 * prepared-divisor quotient the softmax rows use.  out1 may be NULL unless
 * func 7. */
int q48_fp_eval(q48_ctx *ctx, int func, const int64_t *x, const int64_t *y,
                int64_t *out0, int64_t *out1, int n);

/* ---- fused decode ops ------------------------------------------------------- */
/* Each is exactly the composition it names (same bits as the separate ops);
 * fusing removes launches and a round trip of the activation through HBM.
 * With int64 weights an output may share words with the vectors a GEMV reads
 * (not with W): such a call runs as separate launches through a temporary. */

/* y = W . rmsnorm(x, norm_w): rmsnorm (llama_int.c:1048-1058) followed by
 * matmul_vec (llama_int.c:1014-1046), K = dim of x.  Used for q|k|v
 * (llama_int.c:1384-1389) and the lm_head (llama_int.c:2876-2880). */
int q48_rmsnorm_gemv(q48_ctx *ctx, int64_t *y, const int64_t *W, const int64_t *x,
                     const int64_t *norm_w, int M, int K);

/* acc += W . x: matmul_vec then the residual add (llama_int.c:1532-1535,
 * 1553-1556). */
int q48_gemv_residual(q48_ctx *ctx, int64_t *acc, const int64_t *W, const int64_t *x,
                      int M, int K);

/* out[i] = fp_mul(fp_silu(g_i), u_i) with g = rows 0..ffn-1 and u = rows
 * ffn..2ffn-1 of Wgu . rmsnorm(x, norm_w): the post-attention norm, the
 * gate/up projections and SwiGLU (llama_int.c:1544-1552).  Wgu [2*ffn][K]
 * is gate_proj stacked on up_proj. */
int q48_rmsnorm_gemv_swiglu(q48_ctx *ctx, int64_t *out, const int64_t *Wgu,
                            const int64_t *x, const int64_t *norm_w, int ffn, int K);

/* q48_attn_decode with the RoPE of q and k_new fused in (rope_apply,
 * llama_int.c:997-1008, 1392-1395): q and k_new are given unrotated, the
 * cache receives rotated k.  Needs q48_rope_init(head_dim, >= max_seq) and
 * head_dim % 8 == 0. */
int q48_attn_decode_rope(q48_ctx *ctx, int64_t *out, const int64_t *q,
                         int64_t *kcache, int64_t *vcache, const int64_t *k_new,
                         const int64_t *v_new, int layer, int pos, int n_heads,
                         int n_kv, int head_dim, int max_seq);
/* First position at which q48_attn_decode_rope(_prefetch) serves a head with
 * the split kernels (chunks of the cache over many compute units) instead
 * of one block per head.  Kernels are chosen from the pos argument, also in
 * step mode: a graph captured below this position keeps the one-block
 * kernels as replays move past it (same bits, slower). */
int q48_attn_split_min(void);
/* Split attention as ONE launch (on: the default), whose chunk blocks hand
 * the softmax's global max and sum to each other at two barriers inside the
 * kernel, or as three launches (off).  Same bits either way.  The one-launch
 * form serves a cache whose blocks (heads x chunks of max_seq) can all be
 * resident at once; otherwise the three launches run.  No reference
 * counterpart: a scheduling choice of this library. */
int q48_set_attn_one_launch(q48_ctx *ctx, int on);
/* Batched-prefill attention (q48_attn_prefill) with the q.k and p.v products
 * on the int8 matrix cores (on: the default, for head_dim 32, 64 or 128 and
 * up to 16320 cache rows) or on the VALU, one block per (head, query row)
 * (off; up to 4096 cache rows).  Same bits either way.  No reference
 * counterpart: a kernel choice of this library. */
int q48_set_pf_attn_mfma(q48_ctx *ctx, int on);
/* Decode attention from q48_attn_split_min() (the one-launch split form, head_dim
 * 64) with its q.k scores on the int8 matrix cores (on: the default) or on
 * the VALU (off).  Same bits either way.  No reference counterpart: a kernel
 * choice of this library. */
int q48_set_attn_g_mfma(q48_ctx *ctx, int on);
/* q48_attn_decode_rope without any device allocation.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under hipGraph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  q48_attn_decode_rope grows the context's workspace with
 * hipMalloc when a longer cache needs it; this entry takes the split
 * attention's workspace from a fixed per-device array of 4 MiB (its usable
 * part is q48_attn_noalloc_max_bytes()) and returns Q48_ETOOBIG, launching
 * nothing, when the call would need more.  Same arguments, same bits.  Every
 * call on one GPU shares that GPU's array: calls that overlap on one GPU
 * (from two contexts or two streams) race. */
int q48_attn_decode_rope_noalloc(q48_ctx *ctx, int64_t *out, const int64_t *q,
                                 int64_t *kcache, int64_t *vcache, const int64_t *k_new,
                                 const int64_t *v_new, int layer, int pos, int n_heads,
                                 int n_kv, int head_dim, int max_seq);
size_t q48_attn_noalloc_max_bytes(void);
/* Synchronises; Q48_ETIMEOUT if a one-launch split attention launched since
 * the last call could not finish (a block waited past its bound: blocks were
 * not all resident; its output is then wrong and its exchange words are
 * cleared, so the next launch starts clean), else Q48_OK.  The reference's
 * llama_forward cannot fail this way; its callers treat a failed forward
 * (NULL) as the end of generation (llama_int.c:3083-3086, 3106), and
 * q48h_forward / q48h_generate / q48h_decode_* return this code. */
int q48_attn_status(q48_ctx *ctx);
/* The one-launch split attention's wait bound in wall-clock ticks (a
 * negative value restores the default, 2^24 ticks); 0 makes every chunk
 * block give up at its first exchange without waiting, so that the timeout
 * path can be tested while every block still exits normally.  No reference
 * counterpart.  Changes q48_graph_stamp. */
int q48_set_attn_wait(q48_ctx *ctx, int64_t ticks);

/* Long normed GEMVs (more than two rounds of 8-row groups: gate|up, lm_head)
 * run as persistent blocks that loop over row groups (on: the default), or
 * one block per group (off).  Same bits either way.  No reference
 * counterpart: a scheduling choice of this library. */
int q48_set_gemv_persistent(q48_ctx *ctx, int on);
/* q48_attn_decode_rope that also reads [prefetch, prefetch + prefetch_bytes)
 * (16-byte aligned; typically the next op's weights, W_o) on the compute
 * units the heads leave idle, so that the next op finds them in the
 * device-side cache.  No reference counterpart (a scheduling hint: the
 * results are those of q48_attn_decode_rope). */
int q48_attn_decode_rope_prefetch(q48_ctx *ctx, int64_t *out, const int64_t *q,
                                  int64_t *kcache, int64_t *vcache, const int64_t *k_new,
                                  const int64_t *v_new, int layer, int pos, int n_heads,
                                  int n_kv, int head_dim, int max_seq, const void *prefetch,
                                  size_t prefetch_bytes);

/* The decode layer's first half split the other way: the projection's
 * epilogue does RoPE and the KV store, so that attention starts from the
 * cache.  q48_norm_gemv_rope_kv: qkv = W . rmsnorm(x, norm_w) (statistics as
 * partial sums, see Q48_STATS_WORDS; rmsnorm and matmul_vec,
 * llama_int.c:1048-1058, 1014-1046, 1384-1389) with W the q, k and v
 * projections stacked ([(n_heads + 2 n_kv) head_dim][K]), then rope_apply on
 * the q and k heads (llama_int.c:997-1008, 1392-1395) and k, v stored in the
 * caches at pos (llama_int.c:1414-1416).  qkv receives every row, q and k
 * rotated.  Needs q48_rope_init(head_dim, >= max_seq), head_dim 32, 64 or
 * 128.  In step mode pos is read from the device-side state. */
int q48_norm_gemv_rope_kv(q48_ctx *ctx, int64_t *qkv, const int64_t *W, const int64_t *x,
                          const int64_t *norm_w, const int64_t *stats, int64_t *kcache,
                          int64_t *vcache, int layer, int pos, int n_heads, int n_kv,
                          int head_dim, int max_seq, int K);
/* q48_norm_gemv_rope_kv on bfloat16 weights (the bfloat16 section's rules). */
int q48_norm_gemv_rope_kv_bf16(q48_ctx *ctx, int64_t *qkv, const uint16_t *W,
                               const int64_t *x, const int64_t *norm_w, const int64_t *stats,
                               int64_t *kcache, int64_t *vcache, int layer, int pos,
                               int n_heads, int n_kv, int head_dim, int max_seq, int K);
/* Attention of one token over the cache (llama_int.c:1060-1072, 1502-1529)
 * after q48_norm_gemv_rope_kv: q rotated, the key and value at pos already
 * in the caches.  max_seq <= 4096; prefetch (16-byte aligned, may be NULL)
 * as in q48_attn_decode_rope_prefetch.  Same bits as q48_attn_decode_rope on
 * the unrotated inputs. */
int q48_attn_decode_cached(q48_ctx *ctx, int64_t *out, const int64_t *q, int64_t *kcache,
                           int64_t *vcache, int layer, int pos, int n_heads, int n_kv,
                           int head_dim, int max_seq, const void *prefetch,
                           size_t prefetch_bytes);

/* The same fusions with the rmsnorm statistics computed once per vector:
 * r = fp_inv_sqrt((int64)((sum x^2 >> 48) / dim) + 2814749767), the scalar
 * of rmsnorm (llama_int.c:1049-1055), lives in device memory (*r) and the
 * consumers apply fp_mul(fp_mul(x, r), norm_w) (llama_int.c:1056-1057). */
int q48_rms_inv(q48_ctx *ctx, int64_t *r_out, const int64_t *x, int dim);
/* out = table[token] (llama_int.c:2822-2824) and *r_out = its statistics. */
int q48_embed_rms(q48_ctx *ctx, int64_t *out, const int64_t *table, int token, int dim,
                  int64_t *r_out);
/* y = W . (x * r * norm_w): q48_rmsnorm_gemv with r given. */
int q48_norm_gemv(q48_ctx *ctx, int64_t *y, const int64_t *W, const int64_t *x,
                  const int64_t *norm_w, const int64_t *r, int M, int K);
/* q48_rmsnorm_gemv_swiglu with r given. */
int q48_norm_gemv_swiglu(q48_ctx *ctx, int64_t *out, const int64_t *Wgu, const int64_t *x,
                         const int64_t *norm_w, const int64_t *r, int ffn, int K);
/* acc += W . x (residual add), then *r_out = the rmsnorm statistics of the
 * updated acc (dim M): the producer of the next norm's r. */
int q48_gemv_residual_rms(q48_ctx *ctx, int64_t *acc, const int64_t *W, const int64_t *x,
                          int M, int K, int64_t *r_out);

/* The same fusions with the statistics left as partial sums: stats[2i],
 * stats[2i + 1] (lo, hi words) hold the 128-bit sum of squares of rows
 * 8i .. 8i+7 of the vector, Q48_STATS_WORDS(dim) int64 words in all.  The
 * producer of a vector writes them with no cross-block step; every block of
 * the consumer adds them up and derives r itself while its weight loads are
 * in flight (same r, same bits as rmsnorm, llama_int.c:1048-1058). */
#define Q48_STATS_WORDS(dim) (2 * (((dim) + 7) / 8))
int q48_rms_stats(q48_ctx *ctx, int64_t *stats, const int64_t *x, int dim);
/* out = table[token] (llama_int.c:2822-2824) and the partial sums of that row. */
int q48_embed_stats(q48_ctx *ctx, int64_t *out, const int64_t *table, int token, int dim,
                    int64_t *stats);
/* y = W . rmsnorm(x, norm_w) with the statistics of x given as partial sums. */
int q48_norm_gemv_stats(q48_ctx *ctx, int64_t *y, const int64_t *W, const int64_t *x,
                        const int64_t *norm_w, const int64_t *stats, int M, int K);
/* q48_rmsnorm_gemv_swiglu with the statistics of x given as partial sums. */
int q48_norm_gemv_swiglu_stats(q48_ctx *ctx, int64_t *out, const int64_t *Wgu,
                               const int64_t *x, const int64_t *norm_w,
                               const int64_t *stats, int ffn, int K);
/* acc += W . x (residual add), then the partial sums of the updated acc
 * (dim M) into stats. */
int q48_gemv_residual_stats(q48_ctx *ctx, int64_t *acc, const int64_t *W, const int64_t *x,
                            int M, int K, int64_t *stats);

/* ---- bfloat16-resident weights ------------------------------------------
 * The reference's .mgwc format (llama_int.c:1906-1929) keeps weights as
 * their bfloat16 bits and expands them with bfloat16_to_q1648
 * (safetensors.h:115-152) at load.  These GEMVs keep the bits in device
 * memory (2 bytes per weight) and expand each one in the kernel with the
 * same rule, so for weights that are bfloat16 values the results are the
 * int64-weight results, bit for bit, from a quarter of the weight bytes.
 * W is [M][K] uint16, 16-byte aligned; x, norm_w and stats 16-byte aligned;
 * K a multiple of 512 (else Q48_EINVAL).  No reference counterpart beyond
 * the format: the reference expands at load time. */

/* out[i] = the bfloat16 bits b with bfloat16_to_q1648(b) == in[i], for n
 * elements; *inexact = 1 (host int) when some in[i] has no such b (then the
 * weights must stay int64).  Synchronises. */
int q48_bf16_pack(q48_ctx *ctx, uint16_t *out, const int64_t *in, size_t n, int *inexact);
/* q48_gemv on bfloat16 weights. */
int q48_gemv_bf16(q48_ctx *ctx, int64_t *y, const uint16_t *W, const int64_t *x, int M, int K);
/* q48_norm_gemv_stats on bfloat16 weights. */
int q48_norm_gemv_stats_bf16(q48_ctx *ctx, int64_t *y, const uint16_t *W, const int64_t *x,
                             const int64_t *norm_w, const int64_t *stats, int M, int K);
/* q48_norm_gemv_swiglu_stats on bfloat16 weights (Wgu is [2 ffn][K]). */
int q48_norm_gemv_swiglu_stats_bf16(q48_ctx *ctx, int64_t *out, const uint16_t *Wgu,
                                    const int64_t *x, const int64_t *norm_w,
                                    const int64_t *stats, int ffn, int K);
/* q48_gemv_residual_stats on bfloat16 weights. */
int q48_gemv_residual_stats_bf16(q48_ctx *ctx, int64_t *acc, const uint16_t *W,
                                 const int64_t *x, int M, int K, int64_t *stats);

/* ---- device-resident decode steps (graph replay) ---------------------------- */
/* No reference counterpart: llama_int's generate (llama_int.c:3067-3135)
 * passes token and pos as C arguments each call.  In step mode q48_embed,
 * q48_embed_rms and q48_embed_stats read the token, and q48_rope / q48_attn_decode(_rope) read pos, from a
 * device-side state {token, pos, count} instead of their arguments, and
 * q48_argmax_step writes the greedy token back into that state (pos += 1),
 * so one captured forward can be replayed for consecutive tokens with no
 * host round trip.  Kernels ignore a state position outside the cache. */
int q48_step_mode(q48_ctx *ctx, int on);
int q48_step_set(q48_ctx *ctx, int token, int pos);      /* stream-ordered */
int q48_step_get(q48_ctx *ctx, int *token, int *pos, int *count);  /* syncs */
/* argmax (llama_int.c:2888-2893) of v[0..n) into the state; the token is
 * also stored at d_tokens[count] while count < cap. */
int q48_argmax_step(q48_ctx *ctx, const int64_t *v, int n, int *d_tokens, int cap);
/* Parity hook of the replayed steps.  No reference counterpart: it keeps the
 * logits of each step (what llama_forward returns to generate,
 * llama_int.c:3082 and 3105) so that the host can hash every replayed step.
 * Copies v[0..n) to rec[count * n ..] while count < cap, count being the
 * state's number of tokens chosen so far; enqueue it before the step's
 * q48_argmax_step or q48_sample_step. */
int q48_record_step(q48_ctx *ctx, const int64_t *v, int n, int64_t *rec, int cap);
/* q48_record_step (into rec, rec_cap) followed by q48_argmax_step, as one
 * launch: the same record and the same token.  No reference counterpart
 * (as q48_record_step). */
int q48_argmax_record_step(q48_ctx *ctx, const int64_t *v, int n, int *d_tokens, int cap,
                           int64_t *rec, int rec_cap);


/* ---- batched prefill ------------------------------------------------------ */
/* No reference counterpart as a batch: llama_int's prefill calls
 * llama_forward once per prompt token (llama_int.c:3081-3092).  These are the
 * per-token ops of transformer_layer_forward over T rows (token t at
 * position p0 + t), for a prefill whose projections are q48_gemm; each row
 * gets the reference's bits for its token.  Row-major [T][...] buffers. */
/* hidden[t] = embed[d_tokens[t]] (llama_int.c:2822-2824; ids on the device,
 * range-checked by the caller). */
int q48_embed_rows(q48_ctx *ctx, int64_t *H, const int64_t *table, const int *d_tokens, int T,
                   int dim);
/* rmsnorm (llama_int.c:1048-1058) of every row. */
int q48_rmsnorm_rows(q48_ctx *ctx, int64_t *out, const int64_t *X, const int64_t *w, int T,
                     int dim);
/* RoPE (llama_int.c:997-1008, 1392-1395) of the q and k heads of every
 * [q | k | v] row in place, then the KV store (1414-1416) at p0 + t. */
int q48_rope_store_rows(q48_ctx *ctx, int64_t *QKV, int64_t *kcache, int64_t *vcache, int layer,
                        int p0, int T, int n_heads, int n_kv, int head_dim, int max_seq);
/* Exact causal attention (llama_int.c:1433, 1502-1529) of the rotated q of
 * every row over cache positions 0 .. p0 + t (stored by
 * q48_rope_store_rows); out[T][n_heads * head_dim].  p0 + T at most 16320
 * (head_dim 32, 64, 128; 4096 on the VALU kernel, see q48_set_pf_attn_mfma).
 * Uses up to 16 * 8 bytes per (head, query row, cache row) of workspace. */
int q48_attn_prefill(q48_ctx *ctx, int64_t *out, const int64_t *QKV, int64_t *kcache,
                     int64_t *vcache, int layer, int p0, int T, int n_heads, int n_kv,
                     int head_dim, int max_seq);
/* SwiGLU (llama_int.c:1549-1552) of every [gate | up] row: out[T][ffn]. */
int q48_silu_mul_rows(q48_ctx *ctx, int64_t *out, const int64_t *GU, int T, int ffn);

/* ---- quantised key/value cache -------------------------------------------- */
/* The keys and values of a cache as 8- or 4-bit codes with one Q16.48 step per
 * (position, KV head): 1.125 or 0.625 bytes a value of 64-wide heads instead
 * of 8.  A head vector x of head_dim words becomes, with Q = 127 (8 bits) or 7
 * (4 bits) and a = max |x_d|,
 *   step   = min(ceil(a / Q), floor((2^63 - 1) / Q))
 *   code_d = sign(x_d) min(Q, floor((|x_d| + floor(step / 2)) / step)), 0 where
 *            step is 0,
 * and is read as code_d * step (never past 63 bits), at most half a step from
 * x_d (a word more than the step's half where |x_d| > 2^63 - 64).  Attention
 * over the cache is exactly attention over those values.  The reference's own
 * quantised caches (llama_int.c:129-179, 1197-1235) are other formats.
 *
 * The four arrays are device memory of the caller: k and v (16-byte aligned)
 * [layers][max_seq][n_kv][head_dim * bits / 8] bytes, k_step and v_step
 * [layers][max_seq][n_kv].  At 8 bits a code is a signed byte; at 4 bits byte b
 * of a head holds dim b in its low and dim b + head_dim / 2 in its high half,
 * two's complement.  head_dim 32, 64 or 128; max_seq at most 32767 (as
 * q48_rope_init), layers and n_kv at most 65535.  The struct itself is read during
 * the call only. */
typedef struct {
    void *k, *v;
    int64_t *k_step, *v_step;
    int bits;
    int layers, max_seq, n_kv, head_dim;
} q48_qcache;
/* bytes of k (or v) and of k_step (or v_step) for such a cache */
int q48_qcache_bytes(int bits, int layers, int max_seq, int n_kv, int head_dim, size_t *codes,
                     size_t *steps);
/* Quantise rows p0 .. p0 + T - 1 of a layer from K and V, whose rows of n_kv *
 * head_dim words lie ld words apart (so they may be parts of [q | k | v] rows);
 * keys come rotated.  The counterpart of the KV store
 * (llama_int.c:1414-1416). */
int q48_qcache_store_rows(q48_ctx *ctx, const q48_qcache *cache, int layer, int p0, int T,
                          const int64_t *K, const int64_t *V, int ld);
/* The values rows p0 .. p0 + T - 1 stand for, into K and V (rows ld words apart;
 * words between the rows are left as they are). */
int q48_qcache_load_rows(q48_ctx *ctx, int64_t *K, int64_t *V, const q48_qcache *cache, int layer,
                         int p0, int T, int ld);
/* q48_rope_store_rows into a quantised cache: RoPE of the q and k heads of every
 * [q | k | v] row in place, then the quantised store at p0 + t.  d_pos: the
 * rows' RoPE positions (device, T ints; NULL: p0 + t), as drafted tokens of a
 * tree have them.  A row whose position is outside the RoPE tables is neither
 * rotated nor stored.  Needs q48_rope_init(head_dim, >= max_seq). */
int q48_rope_store_rows_qcache(q48_ctx *ctx, int64_t *QKV, const q48_qcache *cache, int layer,
                               int p0, int T, const int *d_pos, int n_heads);
/* q48_attn_decode over a quantised cache: k_new and v_new are quantised into row
 * pos, then rows 0 .. pos are attended to.  Same bits as q48_attn_decode over
 * the values the cache stands for.  In step mode pos is read from the
 * device-side state; the kernels are chosen from the pos argument also then, so a
 * graph captured at a short position stays right, and gets slower, as replays move
 * past it.  The context's workspace (scores, for long spans) reaches its size in the
 * first call of a shape, so call once before capturing.  out shares no words with q,
 * k_new or v_new.  n_heads at most 1024. */
int q48_attn_decode_qcache(q48_ctx *ctx, int64_t *out, const int64_t *q, const q48_qcache *cache,
                           const int64_t *k_new, const int64_t *v_new, int layer, int pos,
                           int n_heads);
/* The same with the RoPE of q and k_new fused in (they come unrotated and stay
 * so), as q48_attn_decode_rope.  Needs q48_rope_init(head_dim, >= max_seq). */
int q48_attn_decode_rope_qcache(q48_ctx *ctx, int64_t *out, const int64_t *q,
                                const q48_qcache *cache, const int64_t *k_new,
                                const int64_t *v_new, int layer, int pos, int n_heads);

/* ---- drafted tokens: attention of rows under a mask ------------------------- */
/* Attention of T rotated rows [q | k | v] over a cache that already holds their
 * keys and values at rows p0 .. p0 + T - 1.  Row t attends to every row before
 * p0 and, among the T new rows, to those its mask names: mask is device memory
 * of ceil(T / 64) 64-bit words a row, bit j % 64 of word j / 64 of row t for
 * row p0 + j (bits from T on are ignored); NULL: rows p0 .. p0 + t, causal.  A
 * row that attends to nothing (p0 = 0, no bit) gives zeros.  Each row's result
 * is the reference's exact attention (llama_int.c:1502-1529) over the rows it
 * attends to, in cache order, so a token of a tree gets the words that decoding
 * its own path gives.  Workspace as for q48_attn_decode_qcache (1 GiB of scores at
 * most, and a thirtieth of that beside them: more rows take several launches).
 * out [T][n_heads * head_dim] shares no words with QKV.
 * head_dim 32, 64 or 128; n_heads at most 1024; p0 + T at most 32767. */
int q48_attn_tree(q48_ctx *ctx, int64_t *out, const int64_t *QKV, const int64_t *kcache,
                  const int64_t *vcache, int layer, int p0, int T, int n_heads, int n_kv,
                  int head_dim, int max_seq, const uint64_t *mask);
int q48_attn_rows_qcache(q48_ctx *ctx, int64_t *out, const int64_t *QKV, const q48_qcache *cache,
                         int layer, int p0, int T, int n_heads, const uint64_t *mask);
/* q48_rope_store_rows with the rows' RoPE positions given (device, T ints): row t
 * is rotated at d_pos[t] and stored at cache row p0 + t.  A row whose position
 * is outside the RoPE tables is neither rotated nor stored. */
int q48_rope_store_rows_at(q48_ctx *ctx, int64_t *QKV, int64_t *kcache, int64_t *vcache,
                           int layer, int p0, int T, const int *d_pos, int n_heads, int n_kv,
                           int head_dim, int max_seq);
/* Keep n of the rows stored from p0 on (the accepted path of a tree) in every
 * layer: row p0 + d_rows[i] moves to p0 + i for i < n in turn, d_rows (device)
 * strictly increasing from 0 on.  A d_rows[i] below i or past the cache moves
 * nothing.  Other rows stay as they are. */
int q48_cache_keep_rows(q48_ctx *ctx, int64_t *kcache, int64_t *vcache, int layers, int p0,
                        const int *d_rows, int n, int n_kv, int head_dim, int max_seq);
int q48_qcache_keep_rows(q48_ctx *ctx, const q48_qcache *cache, int p0, const int *d_rows, int n);

/* ---- log probabilities -------------------------------------------------------- */
/* For each of T rows of logits [T][vocab]: the log probability of token
 * d_tokens[t] (0 where that is not an id of the vocabulary, as for a padded
 * row), the entropy of the row's distribution, and its top_n (0 .. 32, at most
 * vocab) most probable tokens, ties to the lowest id, with their log
 * probabilities.  logp (with d_tokens) and entropy may be NULL, top_ids and
 * top_logp [T][top_n] where top_n is 0, but not all of them.  vocab at most
 * 2^22, T at most 2^30.  The outputs share no words with the logits or the
 * tokens (but top_ids may be d_tokens where top_n is 1).  All in Q16.48: with
 * m = max x, u_i = m - x_i (64 bits, unsigned),
 *   e_i = floor(floor(T_j h 2^-48) 2^-n), u_i = n LN2 + j 2^42 + s, 0 <= s < 2^42,
 *         j <= 44, LN2 = 195103586505167, T_j = round(2^48 e^(-j/64)),
 *         h = C_0 - (s (C_1 - (s (... C_6) >> 48)) >> 48), C_k = round(2^48 / k!)
 *   Z = sum e_i, b the largest with (Z >> b) >= 2^48, z = Z >> b, i = (z >> 42) - 64,
 *   d = (z floor(2^54 / (64 + i)) >> 48) - 2^48,
 *   logZ = b LN2 + round(2^48 log(1 + i/64)) + (d g >> 48),
 *         g = D_1 - (d (D_2 - (... D_8) >> 48) >> 48), D_k = round(2^48 / k)
 *   log probability of i = -(u_i + logZ), at least -2^63
 *   entropy = logZ + floor(2^48 ((sum (e_i u_i >> 48)) >> b) / z).
 * Unlike fp_safe_exp (fp_math.h:739-744), whose value is 0 below e^-10 and off by
 * up to 0.3% above, e_i is within 4 units of 2^-48 of e^-u: the many improbable
 * tokens of a vocabulary count.  Vocabularies past 8192 may use the context's workspace:
 * call once before capturing.  No reference counterpart. */
int q48_logprobs_rows(q48_ctx *ctx, const int64_t *logits, int T, int vocab, const int *d_tokens,
                      int64_t *logp, int64_t *entropy, int top_n, int *top_ids,
                      int64_t *top_logp);

/* ---- sampling (sample_token, llama_int.c:2958-3039) --------------------- */
/* rng_seed (llama_int.c:2909-2920): the xoroshiro128+ state of a seed
 * (SplitMix64), computed on the host.  Upload it to a device buffer of two
 * uint64 words for q48_sample / q48_sample_step. */
void q48_rng_seed(uint64_t seed, uint64_t state[2]);
/* sample_token on device logits[0..vocab): temperature (Q16.48), top_k
 * (0 = off), top_p (Q16.48, ONE = off), and one rng_next draw from the
 * device state rng[2], advanced in place.  Below a temperature of 0.01 it is
 * argmax and draws nothing, as the reference.  The token goes to *token
 * (host; the call synchronises). */
int q48_sample(q48_ctx *ctx, const int64_t *logits, int vocab, int64_t temperature,
               int top_k, int64_t top_p, uint64_t *rng, int *token);
/* The same into the decode-step state (as q48_argmax_step): stream-ordered,
 * graph-capturable once q48_sample_reserve has sized the workspace. */
int q48_sample_step(q48_ctx *ctx, const int64_t *logits, int vocab, int64_t temperature,
                    int top_k, int64_t top_p, uint64_t *rng, int *d_tokens, int cap);
/* Size the sampling workspace for `vocab` logits (synchronises; not during
 * capture). */
int q48_sample_reserve(q48_ctx *ctx, int vocab);

/* Graph capture of stream-ordered ops (no reference counterpart: the
 * reference calls llama_forward once per token, llama_int.c:3103-3113; a
 * captured decode step replays that call's kernels with the token and
 * position read from the device step state).
 *
 * The context graph: begin captures into it (replacing any previous one),
 * end instantiates it, launch replays it, drop destroys it.  Destroying waits
 * for the stream first, so in-flight launches finish. */
int q48_graph_begin(q48_ctx *ctx);
int q48_graph_end(q48_ctx *ctx);
int q48_graph_launch(q48_ctx *ctx, int times);
int q48_graph_drop(q48_ctx *ctx);
/* Graphs the caller holds, any number at once: q48_graph_capture starts a
 * capture that q48_graph_instantiate ends into a new handle (uploaded to the
 * device before it returns); q48_graph_replay launches it `times` times;
 * q48_graph_destroy waits for the stream and frees it.  Workspaces the
 * context replaces while any graph is alive are freed only after the last
 * graph is destroyed, so a graph never replays against freed memory.
 * q48_graph_stamp changes whenever a context setting that selects the
 * kernels or kernel arguments a capture records changes (the q48_set_*
 * switches, q48_rope_init with new parameters): a caller that caches graphs
 * keys them on it. */
typedef struct q48_graph q48_graph;
int q48_graph_capture(q48_ctx *ctx);
int q48_graph_instantiate(q48_ctx *ctx, q48_graph **out);
int q48_graph_replay(q48_ctx *ctx, q48_graph *graph, int times);
int q48_graph_destroy(q48_ctx *ctx, q48_graph *graph);
uint64_t q48_graph_stamp(const q48_ctx *ctx);

/* ---- kernel timing (diagnostic) -------------------------------------------- */

/* HIP-event timing of every GEMV launch (q48_gemv and the fused GEMV entry
 * points) on the context's stream while enabled (no reference counterpart:
 * llama_int's profiler, llama_int.c:65-108, times whole forwards with
 * clock_gettime).  `bytes` is the algorithmic traffic 8*(M*K + K + outputs)
 * per launch.  Not recorded while a graph is being captured. */
typedef struct {
    int launches;
    double ms;       /* sum of launch durations */
    double bytes;    /* sum of algorithmic bytes */
} q48_prof;

int q48_prof_enable(q48_ctx *ctx, int on);
/* Elapsed time of everything enqueued between start and stop, from two HIP
 * events on the context's stream (stop synchronises). */
int q48_timer_start(q48_ctx *ctx);
int q48_timer_stop(q48_ctx *ctx, double *ms);
/* Synchronise, then report (and with reset != 0 clear) the GEMV timings. */
int q48_prof_read(q48_ctx *ctx, q48_prof *gemv, int reset);

#ifdef __cplusplus
}
#endif
#endif /* INTLLM_HIP_H */
