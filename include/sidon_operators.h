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
 * w and bias fp32 [C].  y may be x itself (same stride); any other overlap is
 * refused.  1 <= C <= 8192, C % G == 0.  Statistics and arithmetic in fp32,
 * one rounding at the end.  ws: sidon_group_norm_workspace_bytes bytes, 8-byte
 * aligned, contents irrelevant before and after.
 */
size_t sidon_group_norm_workspace_bytes(int B, int T, int C, int G, int dtype);
int sidon_group_norm_act(const void* x, int64_t ldx, const int32_t* lens, const float* w, const float* bias, float eps,
                         void* y, int64_t ldy, void* ws, size_t ws_bytes, int B, int T, int C, int G, int dtype,
                         int act, sidon_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SIDON_OPERATORS_H */
