/* libtinyinfer_backend.so — entry points with no counterpart in the reference ABI.
 *
 * ti_amd_gemm_i8_fused: the W8A16 linear with the epilogues the GPT-2 runtime
 * fuses into the GEMM (the reference runs them as separate kernels:
 * reference llm/src/runtime.cu:149-153 residual adds, :151 gelu_new):
 *   epilogue 0: y = fp16_rn(acc + bias)
 *   epilogue 1: y = fp16_rn(gelu_tanh(fp16_rn(acc + bias)))
 *   epilogue 2: y = fp16_rn(residual + fp16_rn(acc + bias))   (residual may equal y)
 * a fp16 [M,K], q int8 [K,N], scales fp32 [N], bias fp16 [N] or null, y fp16 [M,N].
 * For callers that want the fused decode/prefill kernels standalone (the
 * configs[1] sweep, tests).  Validation and status codes as ti_v2_gemm_ex_i8. */
#ifndef TINYINFER_AMD_EXT_H
#define TINYINFER_AMD_EXT_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif
int ti_amd_gemm_i8_fused(const uint16_t* a, const int8_t* q, const float* scales,
                         const uint16_t* bias, uint16_t* y, const uint16_t* residual, int m,
                         int n, int k, int epilogue, uintptr_t stream, int device);

/* ti_amd_legacy_gemm_f32_variant: the three FP32 GEMM variants behind
 * ikernels.cuda_bench_matmul(variant, ...) (reference
 * kernels/src/cuda/bench_api.cu:43-51 over kernels/src/cuda/matmul.cu:7-80):
 * 0 naive, 1 LDS-tiled, 2 MFMA-tiled (what ti_cuda_gemm and
 * ti_v2_legacy_gemm_f32 run).  y[M,N] = a[M,K] @ b[K,N] in fp32, device
 * pointers, v2 status codes (3 for an unknown variant). */
int ti_amd_legacy_gemm_f32_variant(int variant, const float* a, const float* b, float* y, int m, int n, int k,
                                   uintptr_t stream, int device);

/* ti_amd_gemm_ex_i8_noalloc: no counterpart in the reference.  For callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc): ti_v2_gemm_ex_i8 with the same
 * arguments, validation, status codes and result bits.  It calls no hipMalloc,
 * hipFree or allocating library routine, and neither does ti_v2_gemm_ex_i8
 * any more: split-K work is finished by the last workgroup of the same launch,
 * with its fp32 partials in static device arrays of the library, one 4 MiB
 * slot per hardware queue (32 slots per GPU, held until the process ends).
 * Limit: a plan is only split when its partials fit the slot (1 Mi floats,
 * 1024 output tiles); larger shapes run unsplit, so no shape is refused.
 * Dispatches on one hardware queue never overlap, so calls on one stream, or
 * on streams that share a queue, do not race, and calls that overlap on
 * different queues use different slots; only with more than 32 hardware
 * queues in use on one GPU can two queues share a slot and overlapping calls
 * on them race. */
int ti_amd_gemm_ex_i8_noalloc(const uint16_t* a, const int8_t* b, const float* scales,
                              const uint16_t* bias, void* y, float* workspace, int m, int n, int k,
                              int dtype, int config, uintptr_t stream, int device);

/* Panel-packed int8 weights for the decode GEMV (M <= 32).  The reference keeps
 * q row-major [K,N] (reference kernels/src/cuda/tc/gemm.cu:21 reads
 * q[r*n + c]); the runtime packs every linear once at load so that each wave
 * load is one contiguous KiB already in MFMA B-operand order:
 *   record (cb, kc) at byte (cb * ceil(K/64) + kc) * 1024, cb = column block of
 *   16, kc = K chunk of 64; lane l's 16 bytes = column cb*16 + (l & 15), rows
 *   kc*64 + 8*(l >> 4) + 0..7 then kc*64 + 32 + 8*(l >> 4) + 0..7; zero past K/N.
 * ti_amd_packed_w8_bytes: size of the packed copy (0 for an invalid shape).
 * ti_amd_pack_w8: device q int8 [K,N] -> packed (16-byte aligned), on `stream`.
 * ti_amd_gemm_w8p_fused: ti_amd_gemm_i8_fused over packed weights, K % 64 == 0,
 * A and packed 16-byte aligned; M <= 32 runs the decode GEMV, M > 32 the
 * multistage MFMA GEMM (64x64 tiles, operands streamed HBM -> LDS with
 * global_load_lds).  Same arithmetic:
 * Y = epilogue(sum_k A[m,k] * fp16_rn(float(q[k,n]) * scales[n]) + bias[n]). */
int64_t ti_amd_packed_w8_bytes(int k, int n);
int ti_amd_pack_w8(const int8_t* q, int k, int n, void* packed, uintptr_t stream, int device);
int ti_amd_gemm_w8p_fused(const uint16_t* a, const void* packed, const float* scales,
                          const uint16_t* bias, uint16_t* y, const uint16_t* residual, int m, int n,
                          int k, int epilogue, uintptr_t stream, int device);

/* Pre-dequantised fp16 weights for the prefill GEMM (M > 32): every weight
 * fp16_rn(float(q[k,n]) * scales[n]) -- the values the int8 kernels compute on
 * the fly (reference kernels/src/cuda/tc/gemm.cu:21,24) -- stored once, so the
 * GEMM is a plain fp16 MFMA GEMM.  Layout: for column block cb (16 columns) and
 * K group kk (32 rows), 1 KiB at (cb * ceil(K/32) + kk) * 1024 bytes, lane l's
 * 16 bytes = column cb*16 + (l & 15), rows kk*32 + 8*(l >> 4) + 0..7; zero past
 * K/N.  ti_amd_packed_w16_bytes: its size; ti_amd_pack_w16: device q int8 [K,N]
 * + scales fp32 [N] -> packed; ti_amd_gemm_w16p_fused: Y = epilogue(A @ W +
 * bias) with the epilogues of ti_amd_gemm_i8_fused, M > 32, K % 32 == 0, A and
 * packed 16-byte aligned. */
int64_t ti_amd_packed_w16_bytes(int k, int n);
int ti_amd_pack_w16(const int8_t* q, const float* scales, int k, int n, void* packed, uintptr_t stream,
                    int device);
int ti_amd_gemm_w16p_fused(const uint16_t* a, const void* packed16, const uint16_t* bias, uint16_t* y,
                           const uint16_t* residual, int m, int n, int k, int epilogue, uintptr_t stream,
                           int device);

/* ti_amd_gemm_w8p_ln_fused: the decode GEMV with the LayerNorm that precedes
 * every GPT-2 linear fed from the residual stream (reference
 * llm/src/runtime.cu:143 ln_1 -> c_attn, :150 ln_2 -> c_fc) computed in its
 * prologue:
 *   Y = epilogue(sum_k LN(A)[m,k] * fp16_rn(float(q[k,n]) * scales[n]) + bias[n]),
 *   LN(A)[m,:] = fp16_rn((A[m,:] * inv - mean * inv) * gamma + beta),
 *   inv = rsqrt(var + eps),
 * mean and var (population, two passes) in fp32 over the K columns of row m,
 * as ti_v2_layernorm_f16 up to fp32 rounding.  The runtime uses it for decode;
 * a caller with many workgroups per row set (the LM head) is better served by
 * one ti_v2_layernorm_f16 pass, since every workgroup normalizes all M rows.  1 <= M <= 32, K % 64 == 0, K <= 2048; A, gamma, beta
 * and packed 16-byte aligned; epilogues as ti_amd_gemm_i8_fused. */
int ti_amd_gemm_w8p_ln_fused(const uint16_t* a, const uint16_t* gamma, const uint16_t* beta, float eps,
                             const void* packed, const float* scales, const uint16_t* bias, uint16_t* y,
                             const uint16_t* residual, int m, int n, int k, int epilogue,
                             uintptr_t stream, int device);

/* FP32 row LayerNorm / last-axis Softmax on a caller stream: the kernels behind
 * ti_cuda_layernorm / ti_cuda_softmax (reference backend/runtime.cpp:10-12),
 * with the v2 conventions (device pointers, stream, device check, status code
 * instead of abort) so they can be ordered with other work or graph-captured.
 * Validation as ti_v2_layernorm_f16 / ti_v2_softmax_f16 with 4-byte alignment. */
int ti_amd_layernorm_f32(const float* x, const float* gamma, const float* beta, float* y,
                         int rows, int cols, float eps, uintptr_t stream, int device);
int ti_amd_softmax_f32(const float* x, float* y, int rows, int cols, uintptr_t stream, int device);
/* y = softmax(LayerNorm(x; gamma, beta, eps)) over the last axis, FP32, one
 * pass per row: the LayerNorm -> Softmax graph that tinyc's norm_softmax issues
 * as ti_cuda_layernorm then ti_cuda_softmax (reference bench/integrated.py:87-92,
 * backend/runtime.cpp:10-12), with the same values as those two calls at half
 * the memory traffic.  Validation as ti_amd_layernorm_f32; y must not overlap x. */
int ti_amd_layernorm_softmax_f32(const float* x, const float* gamma, const float* beta, float* y,
                                 int rows, int cols, float eps, uintptr_t stream, int device);

/* The int8 KV cache: no counterpart in the reference, whose caches are fp16.
 * A row of head_dim fp16 values (one token, one key head) is held as head_dim
 * bytes and one fp32 scale = fp32_rn(max|x| / 127) (so 0 for a row of zeros; NaN
 * for a row with an infinity or NaN, which then reads as NaN); its value is
 * c * scale with c the whole number nearest x / scale, ties to even (0 in a row of zeros).  The caller
 * owns the buffers, all 16-byte aligned: k and v of slots * kv_heads * capacity *
 * head_dim bytes, k_scales and v_scales of slots * kv_heads * capacity floats.
 * Their inner order is the kernels' own (k's rows one after another, v in blocks
 * of 64 tokens).  A call reads the rows that its lengths name: those that were
 * never written count as what the buffers hold (zeros in zeroed ones).
 * capacity is a multiple of 64, head_dim 64 or 128. */
typedef struct ti_amd_kv_i8 {
  uint8_t* k;
  uint8_t* v;
  float* k_scales;
  float* v_scales;
  int32_t slots, kv_heads, capacity, head_dim;
} ti_amd_kv_i8;
/* ti_amd_kv_append_i8: k, v fp16 [batch][kv_heads][rows][head_dim]; row i <
 * lengths[b] (null: every row) becomes token positions[b] + i of slots[b].  The
 * metadata is int32 [batch] on the device.  What lies outside the cache (a slot,
 * a token) is not written; where two requests write the same token the later
 * request's row stays (requests that share a slot look through the later ones, a
 * time that grows with the batch).  batch is at most 65535, rows at most 2^28. */
int ti_amd_kv_append_i8(const ti_amd_kv_i8* cache, const uint16_t* k, const uint16_t* v, const int32_t* slots,
                        const int32_t* positions, const int32_t* lengths, int batch, int rows, uintptr_t stream, int device);
/* ti_amd_kv_read_i8: the same rows back, fp16_rn(fp32(c * scale)); zeros past
 * lengths[b] and outside the cache. */
int ti_amd_kv_read_i8(const ti_amd_kv_i8* cache, uint16_t* k, uint16_t* v, const int32_t* slots, const int32_t* positions,
                      const int32_t* lengths, int batch, int rows, uintptr_t stream, int device);
/* ti_amd_attention_i8kv: q, y fp16 [batch][heads][q_len][head_dim] over the
 * cache; query head h reads key head h / (heads / kv_heads).  Request b's keys
 * are tokens 0 .. kv_lengths[b] - 1 of slots[b] (clamped to the capacity; a slot
 * outside the cache has none).  Query i < q_lengths[b] (null: q_len) sees them
 * all, or with causal = 1 those up to offsets[b] + i; offsets null means
 * kv_lengths[b] - q_lengths[b]: the queries are the request's last tokens.  Rows
 * that see no key, and queries past q_lengths[b], are exactly 0; a row that sees a
 * key or value with an infinity or NaN, or has one in its query, is NaN.  batch and
 * heads are at most 65535, batch * heads * q_len at most 2^23.
 * prefix_len > 0: in front of its own keys every query also sees tokens 0 ..
 * prefix_len - 1 of prefix_slot, whose bytes are read once for the batch (a short
 * prefix of a few requests by each of them).
 * Scores, softmax and sums are fp32; a key's probability times its value's scale is
 * rounded to fp16, relative to what the row itself sees (where few rows share the keys
 * twice: what the first rounding leaves out is added).  How rows and keys are
 * divided follows from the shape arguments, so a request's last bits may differ
 * between batches of other sizes; equal calls give equal bits.
 * max_kv (0: the capacity) is what kv_lengths are expected to stay within: it
 * plans the launch and its workspace, and longer requests are answered too.
 * workspace: ti_amd_attention_i8kv_workspace bytes (-1 for invalid arguments, 0
 * if none is needed), used by this call alone until its work is done. */
int64_t ti_amd_attention_i8kv_workspace(const ti_amd_kv_i8* cache, int batch, int heads, int q_len, int max_kv,
                                        int prefix_len);
int ti_amd_attention_i8kv(const ti_amd_kv_i8* cache, const uint16_t* q, uint16_t* y, const int32_t* slots,
                          const int32_t* kv_lengths, const int32_t* q_lengths, const int32_t* offsets, void* workspace,
                          int64_t workspace_bytes, int batch, int heads, int q_len, int max_kv, int causal,
                          int prefix_slot, int prefix_len, uintptr_t stream, int device);

/* ti_amd_sample: one token per row of logits [batch][vocab] (dtype 0 fp16, 1
 * fp32; batch at most 2^20, vocab 2^18) from uniforms[batch] in [0, 1) (others are taken
 * as the nearest of them, NaN as 0).  Tokens are ordered by logit, ties by
 * index; kept are the first top_k (<= 0: all), of these the shortest run from
 * the front with top_p of their probability (>= 1: all), of these those with at
 * least min_p of the likeliest one's (<= 0: all), the likeliest always.  The
 * token is the first whose cumulative probability among the kept ones exceeds
 * uniforms[b], probs[b] its probability among them.  A temperature that is not
 * above 0, or a logit of +inf, gives the likeliest token with probability 1; a
 * row without a logit above -inf gives 2^31 - 1 with probability 0.  NaN logits
 * are never chosen.  Masses are right to 2^-29 of themselves, and tokens about 32
 * temperatures below the likeliest one, whose weight is e^-32 of its, count as
 * without any (3.4e-9 of it at most, all together).  temperature, top_k, top_p and
 * min_p are per row on the device, or null: then the *_all values hold for every
 * row.  The answer depends on nothing but its row. */
int ti_amd_sample(const void* logits, int dtype, const float* uniforms, const float* temperature, const int32_t* top_k,
                  const float* top_p, const float* min_p, float temperature_all, int top_k_all, float top_p_all,
                  float min_p_all, int32_t* tokens, float* probs, int batch, int vocab, uintptr_t stream, int device);

/* Rotary positions: no counterpart in the reference, whose positions are learned.  A
 * row's first `rotated` dims (even) are turned in pairs, (2 i, 2 i + 1) if interleaved =
 * 1, else (i, rotated / 2 + i): the pair (a, b) of position t becomes amplitude *
 * (a cos w - b sin w, a sin w + b cos w), w = t f_i, in fp32, rounded to fp16 once; the
 * dims behind pass unchanged.  turns holds the frequencies, uint64 [rotated / 2] on the
 * device: turns[i] = 2^64 (f_i / 2 pi mod 1), so angles are exact to 2^-64 of a turn
 * times the position at every int32 position, negative ones too.
 * ti_amd_rotate: x fp16 [batch][heads][rows][dim] with strides in elements (dims
 * contiguous), y contiguous and not overlapping x.  Row i of request b has position
 * positions[b] + i, or positions[b * rows + i] with per_row = 1.  batch and heads are at
 * most 65535, rows * dim at most 2^31. */
int ti_amd_rotate(const uint16_t* x, int64_t x_batch, int64_t x_head, int64_t x_row, uint16_t* y, const int32_t* positions,
                  int per_row, const uint64_t* turns, int rotated, int interleaved, float amplitude, int batch, int heads,
                  int rows, int dim, uintptr_t stream, int device);

/* The paged fp16 KV cache: no counterpart in the reference.  `pages` (16-byte aligned) is
 * page_count pages of kv_heads * 2 * page_size * head_dim values in the kernels' own order; a
 * page is contiguous and may be copied as a whole.  page_size is a power of two from 32 to
 * 1024, head_dim 64 or 128, page_count * kv_heads * page_size at most 2^34.  Which pages hold a
 * request's tokens is the caller's to say: token t of request b lies on page table[b * width +
 * t / page_size] (int32 on the device).  What lies past the table, or on a page outside [0,
 * page_count), does not exist: it is not written, reads as zeros and is not seen. */
typedef struct ti_amd_kv_paged {
  uint16_t* pages;
  int32_t page_count, kv_heads, page_size, head_dim;
} ti_amd_kv_paged;
/* ti_amd_kv_append_paged: k, v fp16 [batch][kv_heads][rows][head_dim] with strides in
 * elements; row i < lengths[b] (null: every row) becomes token positions[b] + i, its key
 * turned by that position if turns is given (rotated a multiple of 16), its value as it
 * is.  With q [batch][heads][rows][head_dim] its rows are turned alike into q_out
 * (contiguous; zeros past lengths[b]; null q: none).  Rows of one call that name one
 * place leave it with the values of either.  batch is at most 65535, rows at most 2^20. */
int ti_amd_kv_append_paged(const ti_amd_kv_paged* cache, const uint16_t* k, int64_t k_batch, int64_t k_head, int64_t k_row,
                           const uint16_t* v, int64_t v_batch, int64_t v_head, int64_t v_row, const uint16_t* q,
                           int64_t q_batch, int64_t q_head, int64_t q_row, uint16_t* q_out, const int32_t* table, int width,
                           const int32_t* positions, const int32_t* lengths, const uint64_t* turns, int rotated,
                           int interleaved, float amplitude, int batch, int heads, int rows, uintptr_t stream, int device);
/* ti_amd_kv_read_paged: the same rows back into contiguous k, v; zeros past lengths[b]. */
int ti_amd_kv_read_paged(const ti_amd_kv_paged* cache, uint16_t* k, uint16_t* v, const int32_t* table, int width,
                         const int32_t* positions, const int32_t* lengths, int batch, int rows, uintptr_t stream, int device);
/* ti_amd_attention_paged: q, y fp16 [batch][heads][q_len][head_dim] over the paged cache;
 * query head h reads key head h / (heads / kv_heads).  Request b's keys are tokens 0 ..
 * kv_lengths[b] - 1, as far as its table reaches.  Query i < q_lengths[b] (null: q_len) sees
 * them all, or with causal = 1 those up to offsets[b] + i; offsets null means kv_lengths[b]
 * - q_lengths[b].  Rows that see no key, and queries past q_lengths[b], are exactly 0.  A row
 * that has an infinity or NaN in its query or sees a NaN in a key is NaN; one that sees an
 * infinity or NaN in a value is not finite in that dim.  A key with a score of -inf (it holds
 * an infinity) has no weight, though an infinity or NaN in its value may count; a row with no
 * other keys is 0.  What a row does not see does not count, whatever memory holds there.
 * Scores, softmax and sums are fp32; a probability is rounded to fp16 for its product.  Where
 * a key head has at most 16 rows (heads / kv_heads * q_len: single tokens of up to 16 heads to
 * a key head) what that rounding leaves out is added; with more rows it is or is not, as the
 * call's extents have it walked.  batch and heads are at most 65535, batch * heads * q_len at
 * most 2^23.
 * max_kv (0: what the table holds) plans the launch and its workspace; longer requests are
 * answered too.  workspace: ti_amd_attention_paged_workspace bytes (-1 for invalid arguments,
 * 0 if none is needed), used by this call alone until its work is done. */
int64_t ti_amd_attention_paged_workspace(const ti_amd_kv_paged* cache, int width, int batch, int heads, int q_len, int max_kv);
int ti_amd_attention_paged(const ti_amd_kv_paged* cache, const uint16_t* q, uint16_t* y, const int32_t* table, int width,
                           const int32_t* kv_lengths, const int32_t* q_lengths, const int32_t* offsets, void* workspace,
                           int64_t workspace_bytes, int batch, int heads, int q_len, int max_kv, int causal, uintptr_t stream,
                           int device);

/* ti_amd_logprobs: of rows of logits [batch][vocab] (dtype 0 fp16, 1 fp32; batch at most
 * 2^20, vocab 2^18) the natural log probabilities of tokens [batch][given] (1 <= given <= 2^16)
 * under the row's softmax, its entropy in nats, and with 0 < top <= 64 its likeliest tokens
 * [batch][top] and their log probabilities (top = 0: both null).  Tokens are ordered by logit,
 * ties by index.  A token outside the vocabulary, or with a logit of -inf or NaN, has the log
 * probability -inf and is no alternative: places left over hold 2^31 - 1 and -inf.  A
 * logit of +inf has all the probability (the first such one).  A row without a logit above -inf
 * has the entropy 0.  Sums are fp32; few rows are read by several workgroups each, which meet in
 * static memory of the library, a slot per hardware queue as for ti_amd_gemm_ex_i8_noalloc: in the
 * last bits they may differ from the same rows in a call of many. */
int ti_amd_logprobs(const void* logits, int dtype, const int32_t* tokens, float* logprobs, float* entropy,
                    float* top_logprobs, int32_t* top_tokens, int batch, int vocab, int given, int top, uintptr_t stream,
                    int device);
#ifdef __cplusplus
}
#endif
#endif
