/*
 * gsq_model -- C ABI of the decoder-glue kernels of the Qwen3.5-hybrid model
 * harness (the model the reference wires in mlx_gsq/models/qwen35.py:11-152).
 *
 * The projections of that model are the packed-weight calls of gsq_b200.h
 * (gsq_qmv / gsq_qmm / gsq_embed).  What lies between them is here: the
 * residual add + RMSNorm, the SwiGLU product, the gated-DeltaNet block
 * (causal depthwise conv, q/k normalisation, decay and write gates, the
 * delta-rule recurrence, the gated RMSNorm), and the single-token GQA
 * attention step.  The reference takes these from mlx_lm (qwen3_5 and
 * gated_delta, not part of the reference repository); the formulas each
 * entry point computes are written beside it.
 *
 * Conventions as in gsq_b200.h: device pointers, asynchronous on `stream`,
 * no allocation, GSQ_OK or a negative gsq_status (gsq_last_error()).
 * Fixed head sizes: gated-DeltaNet key and value heads are 128 wide,
 * attention heads 256 wide (the model's dimensions, qwen35.py:18-25).
 */
#ifndef GSQ_MODEL_H
#define GSQ_MODEL_H

#include "gsq_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* resid[r,:] += delta[r,:] (skipped when delta is NULL), then
 * out[r,:] = resid[r,:] * rsqrt(mean(resid[r,:]^2) + eps) * weight,
 * rounded to out_dtype.  resid, delta, weight fp32; rows x dim. */
GSQ_API int gsq_rmsnorm(float* resid, const float* delta, int64_t rows, int64_t dim, const float* weight, float eps,
                        void* out, int out_dtype, gsq_stream_t stream);

/* out[r,i] = silu(gate[r,i]) * up[r,i] from a [rows, 2n] input of gu_dtype
 * (fp32, fp16 or bf16; computed in fp32): with group == 0 the gate
 * projection's n outputs then the up projection's; with group g > 0
 * (n % g == 0) interleaved groups of g gate then g up outputs (the layout of
 * an interleaved gate|up matrix, see gsq_qmv_swiglu). */
GSQ_API int gsq_silu_mul(const void* gu, int gu_dtype, int64_t rows, int64_t n, int64_t group, void* out,
                         int out_dtype, gsq_stream_t stream);

/* The FFN's gate and up projections and their SwiGLU product in one fused
 * matvec (decode, 0 < rows < 8): `packed` is a packed matrix of 2*n_out rows
 * (K inputs) holding, per 16 rows, 8 rows of ffn_gate then the same 8 rows
 * of ffn_up (n_out % 8 == 0); y[r,i] = silu(gate_i . x_r) * (up_i . x_r),
 * [rows, n_out] in y_dtype -- the down projection's input, with no fp32
 * round trip and no separate kernel.  Arguments and workspace as gsq_qmv
 * for a 2*n_out-row matrix (gsq_qmv_workspace_size(qtype, 2*n_out, K,
 * rows)).  Token counts of 8 and more use gsq_qmm on the same matrix, then
 * gsq_silu_mul with group 8. */
GSQ_API int gsq_qmv_swiglu(int qtype, const void* x, int x_dtype, const uint8_t* packed, int64_t n_out, int64_t K,
                           int64_t rows, void* y, int y_dtype, void* workspace, size_t workspace_bytes,
                           gsq_stream_t stream);

/* Gated-DeltaNet block of T consecutive tokens (the GDN layer of
 * qwen35.py:48-101; nk key heads, nv = multiple of nk value heads, value
 * head h reading key head h % nk).
 *
 *   proj   [T, proj_stride] fp32: columns [0, C) the q|k|v projection
 *          (C = 2*nk*128 + nv*128), columns [C, C + nv*128) the gate z
 *   ab     [T, ab_stride] fp16: columns [0, nv) the decay input a,
 *          [nv, 2nv) the write-gate input b; or NULL, and then the kernel
 *          computes them from x [T, x_stride] fp16 (the layer's normalised
 *          input) and ab_w [2nv, hidden] fp16 (ssm_alpha rows, then
 *          ssm_beta rows) -- one launch fewer for a decode token
 *   conv_state [4, C] fp32: ring of the previous q|k|v inputs, slot p & 3
 *          holding position p's (zeros at the start of a sequence); the T
 *          tokens' inputs are written to their slots
 *   pos    device int32: position of the first of the T tokens
 *   conv_w [C, 4] fp32 depthwise causal taps; A [nv] = -exp(A_log)
 *          (GGUF's ssm_a); dt_bias [nv]; norm_w [128]
 *   state  [nv, 128 (value index j), 128 (key index i)] fp32, updated
 *   scratch  >= gsq_gdn_scratch_bytes(T, nk, nv) bytes (none for T == 1:
 *          one token runs as a single kernel, a CTA per value head)
 *   out    [T, nv*128] in out_dtype
 *
 * Per token: c = silu(conv(q|k|v)); q = rmsnorm(c_q)/128,
 * k = rmsnorm(c_k)/sqrt(128) (no weights, eps 1e-6); g = exp(A *
 * softplus(a + dt_bias)), beta = sigmoid(b); per value head
 * S <- g*S; u = (v - S k) * beta; S <- S + u k^T; o = S q;
 * out = rmsnorm(o) * norm_w * silu(z) (eps). */
GSQ_API size_t gsq_gdn_scratch_bytes(int64_t T, int64_t nk, int64_t nv);
GSQ_API int gsq_gdn(const float* proj, int64_t proj_stride, const uint16_t* ab, int64_t ab_stride,
                    const uint16_t* x, int64_t x_stride, const uint16_t* ab_w, int64_t hidden, int64_t T,
                    int64_t nk, int64_t nv, float* conv_state, const int32_t* pos, const float* conv_w, const float* A,
                    const float* dt_bias, const float* norm_w, float eps, float* state, void* scratch,
                    size_t scratch_bytes, void* out, int out_dtype, gsq_stream_t stream);

/* One decode token of each of `batch` sequences (batched decode), all at
 * position *pos: sequence b's token is row b of proj [batch, proj_stride]
 * and of ab [batch, ab_stride] (or of x [batch, x_stride] with ab NULL); its
 * conv ring is conv_state[b] ([batch, 4, C]), its recurrent state state[b]
 * ([batch, nv, 128, 128]) and its output row b of out [batch, nv*128].  The
 * per-token formulas are gsq_gdn's.  No scratch.  Extends the reference's
 * single-sequence GDN call (mlx_gsq/models/qwen35.py:48-106) to a batch. */
GSQ_API int gsq_gdn_batch(const float* proj, int64_t proj_stride, const uint16_t* ab, int64_t ab_stride,
                          const uint16_t* x, int64_t x_stride, const uint16_t* ab_w, int64_t hidden, int64_t batch,
                          int64_t nk, int64_t nv, float* conv_state, const int32_t* pos, const float* conv_w,
                          const float* A, const float* dt_bias, const float* norm_w, float eps, float* state,
                          void* out, int out_dtype, gsq_stream_t stream);

/* One decode token of gated GQA attention (qwen35.py:137-145 with mlx_lm's
 * attention): qkv [nq*512 + 2*nkv*256] fp32 = per query head 256 query
 * values then 256 gate values, then the key heads, then the value heads.
 * q and k are RMS-normalised per head (q_norm_w, k_norm_w [256], eps), the
 * first `rot` dimensions rotated (rotate-half pairs (d, d + rot/2), angle
 * pos * theta^(-2i/rot)), the key and value stored at row *pos of the caches
 * k_cache / v_cache [max_len, nkv, 256] fp32, and
 * out[h] = softmax(q k^T / 16) v * sigmoid(gate) over positions 0..*pos,
 * rounded to out_dtype ([nq*256]).  pos is a device int32, so that a
 * captured graph replays at the current position; *pos < max_len. */
GSQ_API int gsq_attn_decode(const float* qkv, int64_t nq, int64_t nkv, const float* q_norm_w,
                            const float* k_norm_w, float eps, int64_t rot, float theta, float* k_cache,
                            float* v_cache, int64_t max_len, const int32_t* pos, void* out, int out_dtype,
                            gsq_stream_t stream);

/* gsq_attn_decode for one token of each of `batch` sequences at position
 * *pos: sequence b's qkv is row b of qkv [batch, nq*512 + 2*nkv*256], its
 * caches are k_cache[b] / v_cache[b] ([batch, max_len, nkv, 256]) and its
 * output row b of out [batch, nq*256]. */
GSQ_API int gsq_attn_decode_batch(const float* qkv, int64_t nq, int64_t nkv, const float* q_norm_w,
                                  const float* k_norm_w, float eps, int64_t rot, float theta, float* k_cache,
                                  float* v_cache, int64_t max_len, const int32_t* pos, void* out, int out_dtype,
                                  int64_t batch, gsq_stream_t stream);

/* ---- Quantised key/value cache ------------------------------------------
 * No reference counterpart (the reference keeps mlx_lm's fp16 cache).  The
 * cache of one attention layer is four plain tensors:
 *
 *   codes   [batch, heads, cap, dim] one byte a value, for keys and values:
 *           two's-complement int8 (GSQ_KV_INT8) or e4m3 (GSQ_KV_FP8)
 *   scale   [batch, heads, cap] fp32, for keys and values
 *
 * and a stored vector is code * scale.  With a = max|x| over the vector and
 * m = 127 (int8) or 448 (e4m3), scale = a * (1/m) and code = the nearest (ties
 * to even) of x / scale, with 1/m, scale and the quotient each rounded to fp32
 * (scale downwards where m * scale would pass fp32's range).  A zero vector has
 * scale 0; a vector with an Inf or NaN has scale NaN and codes 0, and reads
 * back as NaN.  Codes that a caller writes by other means must not be e4m3's
 * NaN (0x7f, 0xff) in a position that some row of a call sees.
 * dim is 128 or 256; the codes are 16-byte aligned.
 *
 * Sequence b's new tokens begin at position start[b * start_stride] (device
 * int32; stride 0: one position for all, such as the decode position of a
 * captured graph).  counts (device int32 [batch], or NULL): sequence b has
 * only counts[b] new tokens, the rest of its rows is padding. */
typedef enum { GSQ_KV_INT8 = 0, GSQ_KV_FP8 = 1 } gsq_kv_format;

/* Quantises k and v [batch, tokens, heads, dim] (dtype fp32, fp16 or bf16;
 * strides in elements of the first three dimensions, the last contiguous)
 * into positions start .. start + tokens - 1.  Padding is skipped.  A
 * position outside [0, cap) is not written and sets 3 in gsq_device_status. */
GSQ_API int gsq_kv_append(const void* k, const void* v, int dtype, int64_t batch, int64_t tokens, int64_t heads,
                          int64_t dim, const int64_t* k_strides, const int64_t* v_strides, const int32_t* start,
                          int64_t start_stride, const int32_t* counts, int fmt, void* k_codes, void* v_codes,
                          float* k_scale, float* v_scale, int64_t cap, gsq_stream_t stream);

/* Reads positions start .. start + tokens - 1 back as k and v [batch, tokens,
 * heads, dim] of dtype (code * scale in fp32, rounded once; 16-byte aligned).
 * Padding and positions outside [0, cap) read as zeros. */
GSQ_API int gsq_kv_read(int fmt, const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                        int64_t batch, int64_t heads, int64_t cap, int64_t dim, const int32_t* start,
                        int64_t start_stride, const int32_t* counts, int64_t tokens, void* k, void* v, int dtype,
                        gsq_stream_t stream);

/* gsq_kv_append as the attention layer of the model needs it, from its
 * projection: qkv [batch * tokens, qkv_stride] fp32, per row as in
 * gsq_attn_decode (nq times 256 query and 256 gate values, then keys, then
 * values; heads 256 wide).  Queries and keys are RMS-normalised per head and
 * rotated as there, at positions start + t; the queries go to q [batch,
 * tokens, nq, 256] rounded to fp16, keys and values into the cache.
 * batch * tokens <= 65535. */
GSQ_API int gsq_qkv_append(const float* qkv, int64_t qkv_stride, int64_t batch, int64_t tokens, int64_t nq,
                           int64_t nkv, const float* q_norm_w, const float* k_norm_w, float eps, int64_t rot,
                           float theta, const int32_t* start, int64_t start_stride, void* q, int fmt, void* k_codes,
                           void* v_codes, float* k_scale, float* v_scale, int64_t cap, gsq_stream_t stream);

/* Attention of n new tokens of each sequence, whose keys and values are in
 * the cache already (gsq_kv_append with the same start and counts):
 *
 *   out[b,i,h] = sum_p softmax_p(scale * q[b,i,h] . k[b,p,h']) v[b,p,h']
 *                [* sigmoid(gate[b,i,h])],   h' = h / (heads / kv_heads)
 *
 * over the positions p < cap that row i sees: p <= start + i (a single
 * token, or a chunk of a prompt), or with `tree` the cached text p < start
 * and those new tokens p = start + j, j < counts[b], whose bit j is set in
 * row i of the tree (int32 words [n, ceil(n / 32)] of sequence b at
 * tree + b * tree_stride, bit j % 32 of word j / 32; n <= 1024; stride 0: one
 * tree for all).  A row that sees nothing, and padding, gives zeros.  Scales
 * may have any size; only value scales above 2^57 ask for scores below 2^17.
 *   q     [batch, n, heads, dim] fp16 or bf16, strides in elements of the
 *         first three dimensions; rows 16-byte aligned
 *   gate  fp32 of the same shape with strides of its own, or NULL
 *   out   [batch, n, heads, dim] of q's type, contiguous, 16-byte aligned
 * workspace: gsq_cached_attention_workspace_size() bytes, 256-byte aligned,
 * of any content, for this call alone until it has completed. */
GSQ_API size_t gsq_cached_attention_workspace_size(int64_t batch, int64_t n, int64_t heads, int64_t kv_heads,
                                                   int64_t dim, int64_t cap);
GSQ_API int gsq_cached_attention(const void* q, int dtype, const int64_t* q_strides, int64_t batch, int64_t n,
                                 int64_t heads, int64_t kv_heads, int64_t dim, int fmt, const void* k_codes,
                                 const void* v_codes, const float* k_scale, const float* v_scale, int64_t cap,
                                 const int32_t* start, int64_t start_stride, const int32_t* counts,
                                 const int32_t* tree, int64_t tree_stride, const float* gate,
                                 const int64_t* gate_strides, float scale, void* out, void* workspace,
                                 size_t workspace_bytes, gsq_stream_t stream);

/* ---- Logits --------------------------------------------------------------
 * The history of row r: seen, int32 words [rows, ceil(vocab / 32)] with bit
 * v % 32 of word v / 32 set for every token v of its prompt or output, and
 * counts, int32 [rows, vocab], how often its output holds v (zero wherever
 * the bit is not set).
 *
 * gsq_adjust_logits, per row and token v, each step rounded to fp32:
 *   seen:      z = z > 0 ? z / repetition : z * repetition
 *   counts>0:  z = z - frequency * counts;  z = z - presence
 *   z = z + the sum, in list order, of the row's biases of token v
 *   not allowed: z = -inf
 * out [rows, vocab] fp32 takes z (it may be the logits themselves when they
 * are fp32 with row_stride == vocab); next[r] the token of the row's largest
 * z, the lowest of equal ones (NaN counts as the largest).  With `record`
 * the history learns next[r] as output.
 *   logits      fp32, fp16 or bf16, rows row_stride elements apart
 *   repetition, frequency, presence  device fp32 [rows], or NULL (1, 0, 0);
 *               they need a history
 *   bias_ids, bias_values  [rows, biases], at most 65536; ids outside
 *               [0, vocab) are skipped (padding)
 *   allowed     words like seen's, row r's at r * allowed_stride (0: one mask
 *               for all), bit set = allowed; or NULL
 * rows <= 65535, vocab <= 2^20.  No workspace. */
GSQ_API int gsq_adjust_logits(const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t vocab,
                              int32_t* seen, int32_t* counts, const float* repetition, const float* frequency,
                              const float* presence, const int32_t* bias_ids, const float* bias_values,
                              int64_t biases, const int32_t* allowed, int64_t allowed_stride, float* out,
                              int32_t* next, int record, gsq_stream_t stream);

/* The history of row r learns tokens[r * row_stride + 0 .. n): as output
 * (generated != 0: bit and count) or as prompt (bit only).  Tokens outside
 * [0, vocab) are skipped (padding); a token may come any number of times. */
GSQ_API int gsq_record_tokens(const int32_t* tokens, int64_t row_stride, int64_t rows, int64_t n, int64_t vocab,
                              int32_t* seen, int32_t* counts, int generated, gsq_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GSQ_MODEL_H */
