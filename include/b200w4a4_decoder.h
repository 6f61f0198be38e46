/*
 * b200w4a4_decoder -- C ABI of the decoder-layer operators of libb200w4a4.so: the work around
 * 4-bit linears in a model that reads prompts and answers token by token.
 *
 * Conventions, error codes and dtypes are those of b200w4a4.h: plain device pointers, sizes and a
 * CUDA stream, asynchronous launches on that stream, no allocation, 0 or a negative B200W4A4_E* code.
 * Arguments are checked before anything is launched; a call with nothing to do (M, T, B or Lq = 0)
 * returns 0 and launches nothing.  Pitches are in elements.  Outputs must not overlap inputs
 * unless a declaration says so.
 */
#ifndef B200W4A4_DECODER_H_
#define B200W4A4_DECODER_H_

#include "b200w4a4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* formats of 8-bit codes */
#define B200W4A4_CODES_INT8 0 /* clamp(rint(y / scale), -128, 127), scale = max|y| / 127 * clip */
#define B200W4A4_CODES_E4M3 1 /* y / scale rounded to fp8 e4m3, saturating, scale = max|y| / 448 * clip */

/* Residual addition, RMSNorm and per-token 8-bit codes in one pass:
 *   s = x + residual;  y = s * rsqrt(mean(s^2) + eps) * weight;  codes, scale of y (max|y| >= 1e-5)
 * x, residual [M, D] of x_dtype (F16, BF16, F32), row pitches x_ld / residual_ld; weight [D] of
 * w_dtype; codes [M, D] bytes; scale fp32 [M]; residual_out [M, D] of x_dtype = s rounded once.
 * residual and residual_out are both given or both NULL.  The arithmetic is fp32 and reads s before its
 * rounding; int8 codes are those of the fp32 quotient y / scale, e4m3 codes those of the exact one (decided in 64 bits
 * where fp32 cannot tell two neighbours apart).  1 <= D <= 16384.
 * int8 codes and scales are what b200w4a4_gemm and b200w4a4_linear_w4_group take.
 * A row that is not finite, whose mean(s^2) + eps is below fp32's normal range (and not a row of zeros with
 * eps > 0), or whose scale has no normal reciprocal gets scale NaN and codes 0. */
int b200w4a4_rms_norm_quant(const void* x, int x_dtype, long long x_ld, const void* residual,
                            long long residual_ld, const void* weight, int w_dtype, float eps,
                            void* codes, int code_format, float* scale, void* residual_out, int M,
                            int D, float clip, void* stream);

/* w [N, K] (F16, BF16, F32, contiguous) -> packed u8 [N, K/2] (code 2b in the low nibble, 2b+1 in the
 * high one, two's complement) and scale f16 [N, K/group] = max(absmax, 1e-5) / 7 of each run of
 * `group` values; code = clamp(rint(w / scale), -8, 7).  group: a multiple of 32 that divides K.
 * A group that is not finite, or whose scale passes fp16's range, gets scale NaN and codes 0. */
int b200w4a4_quantize_weight_grouped(const void* w, int w_dtype, void* packed, void* scale, int N,
                                     int K, int group, void* stream);

/* out[m,n] = act_scale[m] * sum_g scale[n,g] * sum_{k in g} x[m,k] * code[n,k] + bias[n]
 * for few tokens (the weight is read once per 8 to 32 of them).  x [M, K] contiguous: F16 or BF16
 * (act_scale NULL), or int8 when x_dtype is B200W4A4_X_INT8 (act_scale fp32 [M]).  packed and
 * scale as b200w4a4_quantize_weight_grouped writes them.  out [M, N] and bias [N] (or NULL) are of
 * out_dtype (F16 or BF16); with out_dtype | B200W4A4_BIAS_F32 the bias is fp32 and added as it is.  Products are
 * exact, sums are fp32 (int32 within a group for int8).
 * M <= 524280, N <= 2^31 - 512, K <= 1048576. */
#define B200W4A4_X_INT8 3
#define B200W4A4_BIAS_F32 16
int b200w4a4_linear_w4_group(const void* x, int x_dtype, const float* act_scale, const void* packed,
                             const void* scale, const void* bias, void* out, int out_dtype, int M,
                             int N, int K, int group, void* stream);

/* Rotary positions on q [T, q_heads, head_dim] and k [T, k_heads, head_dim] (k may be NULL with
 * k_heads 0) in one launch.  dtype F16, BF16 or F32; token and head pitches for each tensor and each
 * output; an output may be its input (same pitches).  cos_sin: fp32 [max_pos, rotary_dim/2, 2];
 * positions: int32 or int64 [T].  interleaved 0: pair i is (i, i + rotary_dim/2); 1: (2i, 2i + 1).
 * Values behind rotary_dim are copied.  inverse 1 rotates back.
 * A token with a negative position is copied unchanged; one at or behind max_pos comes out as NaN in
 * its rotated part.  rotary_dim even, 2 <= rotary_dim <= head_dim <= 512. */
int b200w4a4_rotary(const void* q, long long q_tok, long long q_head, void* q_out, long long qo_tok,
                    long long qo_head, int q_heads, const void* k, long long k_tok, long long k_head,
                    void* k_out, long long ko_tok, long long ko_head, int k_heads, int dtype,
                    const float* cos_sin, long long max_pos, const void* positions, int positions_int64,
                    long long T, int head_dim, int rotary_dim, int interleaved, int inverse, void* stream);

/* Bytes of workspace b200w4a4_window_attention needs for these sizes on the current device (0: none). */
size_t b200w4a4_window_attention_workspace_bytes(int B, int Lq, int Lk, int q_heads, int k_heads,
                                                 int head_dim, int window, int sinks);

/* Causal attention with a sliding window and `sinks` first keys that stay visible.
 * q [B, Lq, q_heads, head_dim], k / v [B, Lk, k_heads, head_dim], dtype F16 or BF16, pitches for batch,
 * token and head (multiples of 8, 16-byte aligned bases), head_dim 64 or 128, q_heads a multiple of
 * k_heads (at most 64 times it).  kv_lens: int32 [B] valid keys of each sequence (NULL: Lk; clamped to
 * 0..Lk).  Query i of a sequence is at position p = kv_len - Lq + i and sees keys j <= p with
 * j > p - window or j < sinks.  out [B, Lq, q_heads, head_dim] contiguous; lse fp32 [B, q_heads, Lq] or
 * NULL (natural log; what b200w4a4_attn_merge takes).  A query that sees nothing: out 0, lse -inf.
 * Keys that no query can see may hold anything; a value that is not finite reaches only the queries that see its key.
 * The softmax weights are rounded to dtype for their product with v, all else is fp32.  window >= 1, sinks >= 0, scale > 0.
 * workspace: of the size above, 16-byte aligned, not shared by calls that may overlap.
 * Calls with 128 queries or more wait on barriers inside the kernel, each for at most a second; one that runs out
 * leaves 106 in the device status word (b200w4a4_last_device_status), and rows of out unwritten. */
int b200w4a4_window_attention(const void* q, long long q_b, long long q_tok, long long q_head,
                              const void* k, long long k_b, long long k_tok, long long k_head,
                              const void* v, long long v_b, long long v_tok, long long v_head,
                              const int* kv_lens, void* out, float* lse, int dtype, int B, int Lq, int Lk,
                              int q_heads, int k_heads, int head_dim, int window, int sinks, float scale,
                              void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* B200W4A4_DECODER_H_ */
