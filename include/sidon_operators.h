/*
 * sidon_operators.h -- C ABI of the operators of large language models beside
 * the encoder's own (MI355X / gfx950), in the same library as sidon_flexrel.h
 * and under the same conventions (device pointers owned by the caller, work
 * enqueued on `stream` with no host synchronisation and no allocation,
 * SIDON_OK or a negative SIDON_E_* code, sidon_last_error()).  None of them
 * has a counterpart in the reference.
 */
#ifndef SIDON_OPERATORS_H
#define SIDON_OPERATORS_H

#include <stddef.h>

#include "sidon_flexrel.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the tensors below. */
#define SIDON_FP32 0
#define SIDON_FP16 1
#define SIDON_BF16 2

/* Activations of the functions below (not every one takes every activation). */
#define SIDON_ACT_NONE 0
#define SIDON_ACT_SILU 1
#define SIDON_ACT_GELU 2 /* 0.5 v (1 + erf(v / sqrt 2)) */
#define SIDON_ACT_RELU 3

/*
 * Group norm with an activation, channels last, over B items of T rows:
 *
 *   y[b, t, c] = act((x[b, t, c] - mean_bg) * rsqrt(var_bg + eps) * w[c] + bias[c]),   g = c / (C / G)
 *
 * with mean and (biased) variance over the C / G channels of group g and the
 * item's valid rows t < lens[b] (int32 [B] on the device, clamped to [0, T];
 * NULL = T).  Rows t >= lens[b] take no part in the statistics, whatever they
 * hold, and are written as zeros.
 *
 * x [B*T, C] and y [B*T, C] of `dtype`, rows ldx / ldy elements apart (>= C);
 * w and bias fp32 [C].  y may be x itself (same stride); any other overlap of y, or of
 * a workspace that the call uses, with another operand is refused.  B <= 65535, T <= 2^30, 1 <= C <= 8192, C % G == 0.  Statistics and arithmetic in fp32,
 * one rounding at the end.  ws: sidon_group_norm_workspace_bytes bytes, 8-byte
 * aligned, contents irrelevant before and after.
 */
size_t sidon_group_norm_workspace_bytes(int B, int T, int C, int G, int dtype);
int sidon_group_norm_act(const void* x, int64_t ldx, const int32_t* lens, const float* w, const float* bias, float eps,
                         void* y, int64_t ldy, void* ws, size_t ws_bytes, int B, int T, int C, int G, int dtype,
                         int act, sidon_stream_t stream);
/* How the two-launch way cuts these sizes, with vectors of `vec` elements (16 bytes, or 1 where the tensors do
 * not lie on them): groups per column block (the last block may have fewer), row chunks per item, and the LDS
 * bytes of a workgroup of the first launch.  No GPU needed. */
int sidon_group_norm_passes(int B, int T, int C, int G, int dtype, int vec, int* block_groups, int* chunks,
                            int* lds_bytes);

/*
 * A shared projection with a low-rank adapter per request.  For row m of
 * x [M, K], with e = ids[m / (M / items)] (int32 [items] on the device):
 *
 *   sidon_adapter_linear     y[m] = act(x[m] . w^T + bias + scale[e] (x[m] . a[e]^T) . b[e]^T)
 *   sidon_adapter_residual   y[m] = add[m] + x[m] . w^T + scale[e] (x[m] . a[e]^T) . b[e]^T
 *
 * Items are M / items consecutive rows each: utterances of a padded batch, or
 * (items == M) single tokens.  An e outside [0, adapters) means no adapter: the
 * row's low-rank term is left out, and no other row's adapter touches it.
 *
 * x [M, K], w [N, K], a [adapters, R, K], b [adapters, N, R] and bias [N] (or NULL)
 * of `dtype` (SIDON_FP16 or SIDON_BF16), K contiguous, rows of x and w ldx / ldw
 * apart, a and b contiguous; scale fp32 [adapters].  linear: y [M, N] of `dtype`,
 * act SIDON_ACT_NONE or SIDON_ACT_SILU.  residual: y and add fp32 [M, N], y may be
 * add itself (same stride), any other overlap of y or of ws with an input is refused.
 * N and K multiples of 64, R a multiple of 8 in [8, 128], M a multiple of items;
 * strides multiples of 8 (y and add of residual: 4); x and w each under 4 GiB;
 * pointers 16-byte aligned (bias 8, ids and scale 4).
 *
 * Sums in fp32.  linear rounds scale (x . a^T) to `dtype` in front of the product
 * with b; residual, whose result is fp32, keeps all of it (two or three summands).
 * fp16 holds them divided by a power of two of each row's own, exactly, so that
 * products past 65504 do not overflow and small ones keep their digits, down to 2^-24
 * of the row's largest.  A row with a product that is no
 * finite number below 2^127 gives infinities or NaN, in that row alone.
 * ws: sidon_adapter_workspace_bytes bytes, 16-byte aligned, contents irrelevant.
 */
size_t sidon_adapter_workspace_bytes(int M, int R, int residual, int dtype);
int sidon_adapter_linear(const void* x, int ldx, const void* w, int ldw, const void* bias, const void* a, const void* b,
                         const float* scale, const int32_t* ids, void* y, int ldy, void* ws, size_t ws_bytes, int M,
                         int N, int K, int R, int adapters, int items, int act, int dtype, sidon_stream_t stream);
int sidon_adapter_residual(const void* x, int ldx, const void* w, int ldw, const void* a, const void* b,
                           const float* scale, const int32_t* ids, const float* add, int ldadd, float* y, int ldy,
                           void* ws, size_t ws_bytes, int M, int N, int K, int R, int adapters, int items, int dtype,
                           sidon_stream_t stream);

/*
 * Differential attention: the difference of two softmax maps over one set of
 * values, with a learned weight per head.  For batch b, head h and query i:
 *
 *   o = sum_j softmax_j(q1 . k1_j / sqrt D) v_j - lambda sum_j softmax_j(q2 . k2_j / sqrt D) v_j
 *   lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lam_init
 *   out = o                                                              norm_w == NULL
 *   out = (1 - lam_init) * norm_w * o / sqrt(mean(o^2) + eps)            otherwise
 *
 * over the keys j < LK = lens[b] (int32 [B] on the device, clamped to [0, S];
 * NULL = S) and, if causal != 0, j <= LK - L + i: the L queries are the last L
 * of the LK positions.  A query that sees no key gives zeros.  Keys and values
 * past LK are not read.  Heads h / (H / Hk) share keys and values.
 *
 * q [B, H, 2, L, D], k [B, Hk, 2, S, D], v [B, Hk, S, 2 D], out [B, H, L, 2 D] of
 * `dtype` (SIDON_FP16 or SIDON_BF16), the last dimension contiguous, the other
 * strides int64 arrays in elements ((batch, head, map, row) for q and k, (batch,
 * head, row) for v and out), multiples of 8 from 0 to 2^40, rows of k and v less
 * than 2^25 apart; D 64 or 128.  lam fp32 [lam_heads, 4, D]: lq1, lk1, lq2, lk2,
 * lam_heads 1 or H.  norm_w fp32 [2 D], eps > 0 with it.  out's rows must not overlap one
 * another, and the memory from its first to its last element must hold nothing of
 * an input; neither must ws.
 *
 * Scores, softmax statistics, sums and the norm in fp32; scores |q . k| / sqrt D up to
 * 2^24 (their fp32 steps past it are more than the softmax takes).  Probabilities are
 * rounded to `dtype` in front of the product with v: each off by half a step of itself,
 * in fp16 down to 2^-23 of the row's largest, and none below 2^-34 of it.  With H / Hk * L
 * <= 32 what the rounding left is multiplied too, and the result is off by its own
 * rounding; with more it may be or not, as the kernel that is fastest for B, L, S and the
 * device has it, so the same prompt can be rounded differently in another batch.  One
 * rounding at the end.  A query that is no number (or whose scores are none) gives NaN
 * and reaches no other.  What a key within LK but past a query's own position holds must
 * be finite (its weight is 0).  ws:
 * sidon_diff_attention_workspace_bytes bytes for these sizes on the current
 * device (0: ws may be NULL), 16-byte aligned, contents irrelevant.
 */
size_t sidon_diff_attention_workspace_bytes(int B, int H, int Hk, int L, int S, int D);
int sidon_diff_attention(const void* q, const void* k, const void* v, const float* lam, int lam_heads, float lam_init,
                         const int32_t* lens, const float* norm_w, float eps, void* out, void* ws, size_t ws_bytes,
                         int B, int H, int Hk, int L, int S, int D, int causal, int dtype, const int64_t* q_strides,
                         const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                         sidon_stream_t stream);

/*
 * The norm of queries and keys for each head, with the position rotation in the
 * same pass.  For a row x of D values (a head of one token) at place p:
 *
 *   y = R_p (w * x / sqrt(mean(x^2) + eps))
 *
 * R_p turns pairs of the first `rot` values by the angle of row p of the tables cos
 * and sin (fp32 [places, rot / 2]): pair j is (j, j + rot / 2), or with interleaved
 * != 0 (2 j, 2 j + 1), and becomes (a cos - b sin, a sin + b cos).  rot == 0: no
 * rotation, tables may be NULL.  The place of token l of item b is pos[b * L + l]
 * (int32 on the device; NULL: l, at most `places` tokens).  A token at a negative
 * place is padding: whatever it holds, its rows become zeros and it has no part in
 * any gradient.  One at a place past the tables gives NaN in what is rotated.
 *
 * q [B, H, L, D] and k [B, Hk, S, D] (Hk == 0: no k) of `dtype` with q_out and k_out
 * of the same shapes; strides int64 arrays (batch, head, row) in elements, multiples
 * of 16 bytes from 0 to 2^40, the last dimension contiguous.  D a multiple of 16 in
 * [16, 256], rot one in [0, D]; q_w and k_w fp32 [D]; eps > 0.  q_out may be q itself
 * (same strides) and k_out k, as column blocks of one tensor too; any other memory
 * that an output shares with another operand is refused, as are outputs whose rows
 * overlap.  Arithmetic in fp32, one rounding at the end; rows whose squares leave fp32
 * are scaled by a power of two.
 *
 * sidon_qk_norm_rotary_bwd: from the gradients dq_out, dk_out of the outputs (any
 * strides as above, 0 too) and the inputs q, k (not the outputs), the gradients dq, dk of
 * `dtype` and dq_w, dk_w fp32 [D], which are written, not added to, and summed in the
 * same order every time.  dq may be dq_out or q itself, dk dk_out or k.  ws:
 * sidon_qk_norm_rotary_workspace_bytes bytes, 16-byte aligned, contents irrelevant.
 */
int sidon_qk_norm_rotary(const void* q, const void* k, void* q_out, void* k_out, const float* q_w, const float* k_w,
                         const float* cos, const float* sin, int places, int rot, int interleaved,
                         const int32_t* q_pos, const int32_t* k_pos, float eps, int B, int H, int Hk, int L, int S, int D,
                         int dtype, const int64_t* q_strides, const int64_t* k_strides, const int64_t* q_out_strides,
                         const int64_t* k_out_strides, sidon_stream_t stream);
size_t sidon_qk_norm_rotary_workspace_bytes(int B, int H, int Hk, int L, int S, int D);
int sidon_qk_norm_rotary_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k, void* dq, void* dk,
                             float* dq_w, float* dk_w, const float* q_w, const float* k_w, const float* cos,
                             const float* sin, int places, int rot, int interleaved, const int32_t* q_pos,
                             const int32_t* k_pos, float eps, void* ws, size_t ws_bytes, int B, int H, int Hk, int L,
                             int S, int D, int dtype, const int64_t* dq_out_strides, const int64_t* dk_out_strides,
                             const int64_t* q_strides, const int64_t* k_strides, const int64_t* dq_strides,
                             const int64_t* dk_strides, sidon_stream_t stream);

/*
 * Attention over states of another length (a decoder's tokens over the encoder's
 * frames).  For batch b, head h and query i < LQ = q_lens[b]:
 *
 *   out = sum_j softmax_j(scale q . k_j) v_j,    lse = log(sum_j exp(scale q . k_j))
 *
 * over the keys j < LK = lens[b] (both int32 [B] on the device, clamped to [0, S] and
 * [0, L]; NULL = S, L).  A query that sees no key, and those from LQ on, whatever they
 * hold, give zeros and an lse of -infinity.  Keys and values past LK are not read.
 * Heads h / (H / Hk) share keys and values.
 *
 * q [B, H, L, D], k and v [B, Hk, S, D], out [B, H, L, D] of `dtype` (SIDON_FP16 or
 * SIDON_BF16), the last dimension contiguous, the other strides int64 arrays (batch,
 * head, row) in elements, multiples of 8 from 0 to 2^40, rows of k and v less than 2^25
 * apart; D 64 or 128; 0 < scale <= 2^100.  lse fp32 [B, H, L] contiguous, or NULL.  out's
 * rows must not overlap one another, and out, lse and ws hold nothing of another operand
 * (out may be a column block of one tensor with q, or lie in turn with it).
 *
 * Scores, softmax statistics and sums in fp32; |scale q . k| up to 2^24.  Probabilities
 * are rounded to `dtype` in front of the product with v: each off by half a step of
 * itself, in fp16 down to 2^-23 of the row's largest, and none below 2^-34 of it.  With
 * H / Hk * L <= 32 what the rounding left is multiplied too, and the result is off by
 * its own rounding; with more it may be or not, as the kernel that is fastest for the
 * sizes and the device has it.  One rounding at the end.  lse sums what was not rounded.
 * A query that is no number gives NaN; another's sum of probabilities may be added up in another order
 * beside it, which is a step of its result at most, and nothing else reaches another.  ws:
 * sidon_cross_attention_workspace_bytes bytes for these sizes on the current device
 * (0: ws may be NULL), 16-byte aligned, contents irrelevant.
 *
 * sidon_cross_attention_bwd: the gradients dq [B, H, L, D], dk and dv [B, Hk, S, D] of
 * `dtype` from the output's, dout, and the forward call's q, k, v, out and lse under the
 * same lens, q_lens and scale; written, not added to; zeros past LQ and LK.  Rows of
 * dout and q less than 2^25 apart, S <= 2^24, B * H <= 2^20, the rest as above; an output
 * may be a column block of one tensor with another operand, or lie in turn with it, and shares
 * no memory.  What dout holds past LQ does not matter.  Products in
 * `dtype` with fp32 sums: probabilities and dS are rounded once in front of them.  fp16
 * scales both by powers of two, so that neither overflows whatever the size of dout.  P keeps
 * its digits down to 2^-29 and vanishes below 2^-40; dS does so down to 2^-28 and 2^-39 of 2 |dout| |v|, with
 * the longest v of the item's key head, and dout of the query itself for dq, the longest of all heads
 * that share the key for dk: what rows a million times shorter than others add there loses digits.
 * sum_j P dP, the number that dS holds the distance from, is taken in fp32 over the keys, not from the
 * rounded out, so that dS is right to its own rounding where one key has nearly all of P.
 * P is formed anew from lse, off by what fp32 leaves of it, some 2^-21 |lse| of itself; |scale q . k| up to 2^20
 * here.  The same bits every time.  ws: sidon_cross_attention_bwd_workspace_bytes bytes.
 */
size_t sidon_cross_attention_workspace_bytes(int B, int H, int Hk, int L, int S, int D);
int sidon_cross_attention(const void* q, const void* k, const void* v, const int32_t* lens, const int32_t* q_lens,
                          float scale, void* out, float* lse, void* ws, size_t ws_bytes, int B, int H, int Hk, int L,
                          int S, int D, int dtype, const int64_t* q_strides, const int64_t* k_strides,
                          const int64_t* v_strides, const int64_t* o_strides, sidon_stream_t stream);
size_t sidon_cross_attention_bwd_workspace_bytes(int B, int H, int Hk, int L, int S, int D, int dtype);
int sidon_cross_attention_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                              const float* lse, const int32_t* lens, const int32_t* q_lens, float scale, void* dq,
                              void* dk, void* dv, void* ws, size_t ws_bytes, int B, int H, int Hk, int L, int S, int D,
                              int dtype, const int64_t* g_strides, const int64_t* q_strides, const int64_t* k_strides,
                              const int64_t* v_strides, const int64_t* o_strides, const int64_t* dq_strides,
                              const int64_t* dk_strides, const int64_t* dv_strides, sidon_stream_t stream);

/*
 * A projection with 4-bit weights and group scales, for few rows:
 *
 *   y[m, n] = act(bias[n] + sum_g s[n, g] sum_{k in g} x[m, k] (w[n, k] - z[n, g]))
 *
 * x [M, K], bias [N] (or NULL) and y [M, N] of `dtype` (SIDON_FP16 or SIDON_BF16), rows
 * ldx (a multiple of 8) and ldy elements apart; x 16-byte aligned, bias and y 2-byte.  act
 * SIDON_ACT_NONE or SIDON_ACT_SILU.  group 32, 64 or 128, K a multiple of it; M <= 2^21,
 * N <= 2^24, K <= 2^20.  y shares no memory with an operand (it may be a column block
 * of one tensor with x).  Sums in fp32, one rounding at the end; a row's sums of |x|
 * over a group times 143 must be fp32 numbers.  A row that holds an infinity or a NaN gives infinities
 * or NaN in all of its outputs, and no other row does.
 *
 * The weights w (0 to 15) and (s, z) as they are laid out once, for N and K rounded up
 * to 16 and 128 with zeros, 16-byte aligned:
 *   words   [N / 16][K / 128][4 q][16 r][4 i] of 32 bits: rows n = 16 t + r, and the inputs
 *           k = 128 b + 32 i + 8 q + (0 2 4 6 1 3 5 7), a nibble each from the lowest
 *   scales  [N / 16][K / 128][128 / group][16 r] of 32 bits: s of `dtype` in the low half, in the
 *           high half what goes off the weight as the kernel has it, of `dtype`: z - 8 in
 *           fp16 (with zeros == 0 taken as 0: z = 8 throughout), 128 + z in bf16
 */
int sidon_int4_linear(const void* x, int64_t ldx, const void* words, const void* scales, const void* bias, void* y,
                      int64_t ldy, int M, int N, int K, int group, int zeros, int act, int dtype,
                      sidon_stream_t stream);
/* How a call of these sizes is cut on the current device (256 compute units without one): tiles of 16 rows and of
 * 16 outputs of a wavefront, wavefronts that K is split over. */
int sidon_int4_linear_tiles(int M, int N, int* rows, int* outputs, int* splits);

#ifdef __cplusplus
}
#endif

#endif /* SIDON_OPERATORS_H */
