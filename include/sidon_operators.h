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

#ifdef __cplusplus
}
#endif

#endif /* SIDON_OPERATORS_H */
