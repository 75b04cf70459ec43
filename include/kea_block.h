/*
 * kea_block.h - the operators of a transformer layer with 8-bit weights in libkea_hip.so (MI355X / gfx950): the int8 x int8
 * matrix product, the norms before and after a block, and attention within a sliding window.
 *
 * Conventions as in kea_lowbit.h: device pointers, int64 sizes and strides (in elements), a hipStream_t as void*,
 * KEA_OK / negative KEA_E* (nothing launched) / positive hipError_t, message in kea_last_error(). No allocation, no
 * host synchronisation: every entry point can be captured into a HIP graph. The reference has no counterpart of these.
 */
#ifndef KEA_BLOCK_H
#define KEA_BLOCK_H

#include <stdint.h>

#include "kea_lowbit.h"

#ifdef __cplusplus
extern "C" {
#endif

/* An element type beside KEA_F32 / KEA_F16 / KEA_BF16, for kea_int8_gemm's y: the raw int32 sums. */
#define KEA_I32 3

/* int8 x int8 matrix product with a scale for each row of q (token) and each row of w (channel):
 *   acc[m][n] = sum_k q[m*ldq + k] * w[n*ldw + k]                     (exact int32: k <= 131071)
 *   y_dtype KEA_I32: y[m*ldy + n] = acc; qs, wscale, bias, residual and flags are not used (pass NULL and 0)
 *   otherwise        r = f(acc) * qs[m]                               (f: int32 -> fp32, to nearest)
 *                    r = bias ? fma(r, wscale[n], bias[n]) : r * wscale[n]
 *                    r = r / (1 + exp(-r))                            with KEA_FLAG_SILU
 *                    y[m*ldy + n] = RN(residual ? residual[m*ldr + n] + r * factor : r)     in y_dtype
 * which is kea_lowbit_gemm's epilogue of one part, so q and qs are what kea_quantize gives with one part.
 *   q, w       rows of 16-byte aligned starts (pointers and ldq, ldw multiples of 16; ldq, ldw >= k). Bytes at k and
 *              behind take no part in the sums, whatever they hold; no byte from the last row's k, rounded up to 16, on
 *              is read.
 *   qs, wscale KEA_F32 or KEA_F16; bias NULL or KEA_F32 / KEA_F16; each aligned to its element size.
 *   residual   NULL or FP32 [m][ldr]; y may be the residual itself (y_dtype KEA_F32, ldy == ldr) and overlaps no other
 *              operand. */
int kea_int8_gemm(const int8_t *q_dev, int64_t ldq, const void *qs_dev, int qs_dtype, const int8_t *w_dev, int64_t ldw,
                  const void *wscale_dev, int ws_dtype, const void *bias_dev, int bias_dtype, void *y_dev, int y_dtype,
                  int64_t ldy, const float *residual_dev, int64_t ldr, float factor, int64_t m, int64_t n, int64_t k,
                  int flags, void *stream);

/* Kinds of norms, and of what a gate passes through. */
#define KEA_NORM_NONE 0
#define KEA_NORM_LAYER 1    /* (v - mean) / sqrt(var + eps) * w + b, var = mean (v - mean)^2 */
#define KEA_NORM_RMS 2      /* v / sqrt(mean v^2 + eps) * w */
#define KEA_GATE_PLAIN 0
#define KEA_GATE_SIGMOID 1
#define KEA_GATE_TANH 2

/* One norm: w and b hold d elements of `dtype` (KEA_F32 / KEA_F16 / KEA_BF16), either may be NULL (1 and 0). */
typedef struct {
    int kind, dtype;
    const void *w_dev, *b_dev;
    float eps;
} kea_norm;

/* The norms behind one block and before the next, with the block's gate and residual scale, in one pass over the rows:
 *   p = post(block[r]);  y[r] = x[r] + factor * act(gate[r / gate_rows]) * p;  z[r] = pre(y[r])
 * for rows r = 0 .. m-1 of d elements, every step in FP32 (a row's mean and variance too) and y and z rounded once, each on
 * its own: z is the norm of y before its rounding. x and y are of x_dtype; block, gate and z of block_dtype.
 *   gate       NULL (1), or [ceil(m / gate_rows)][ldg]: gate_rows rows in turn share a gate row.
 *   y          y may be x itself (in place, ldy == ldx), or the block, and overlaps no other operand. block NULL: y is not
 *              written (pass NULL) and z = pre(x).
 *   z          NULL, or [m][ldz] of block_dtype (pre.kind must not be KEA_NORM_NONE).
 *   q, qs      NULL, or instead of z its quantization to int8 rows with an FP32 scale each, as kea_quantize makes one part:
 *              s = max(max|z| / 127, 1e-30), q = rint(z / s), zero from d to ldq; q [m][ldq], ldq >= d, qs [m].
 * 1 <= d <= 32768. Pointers are aligned to their element size. */
int kea_block_norm(const void *x_dev, int x_dtype, int64_t ldx, const void *block_dev, int block_dtype, int64_t ldb,
                   int64_t m, int64_t d, const kea_norm *post, const void *gate_dev, int64_t ldg, int64_t gate_rows,
                   int gate_act, float factor, void *y_dev, int64_t ldy, const kea_norm *pre, void *z_dev, int64_t ldz,
                   int8_t *q_dev, int64_t ldq, float *qs_dev, void *stream);

/* A tensor [batch][t][heads][d] by its strides in elements; rows of d are contiguous. */
typedef struct {
    void *data_dev;
    int64_t batch_stride, t_stride, head_stride;
} kea_heads;

/* Attention within a sliding window and to the first tokens. Query i (0 <= i < tq) of sequence b stands at position
 * p = q_starts[b] + i among the sequence's keys 0 .. len-1, len = kv_lengths[b] clamped to 0 .. tk, and sees key j < len iff
 *   j <= p + right  and  (j >= p - left  or  j < sinks);
 *   out_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys it sees, 0 where it sees none (or scores of -infinity
 *   alone) or p is outside 0 .. len-1.
 * Head h reads key head h / (heads / kv_heads). A key that a query does not see has no part in its output, whatever k and v
 * hold there; k and v at len and behind are not read. Scores, their maximum and sum and the output's sums are FP32; with
 * KEA_F16 and KEA_BF16 the weights exp(s - max) are rounded to the type, in their sum as in the product with v.
 *   dtype        of q, k, v and out: KEA_F32, KEA_F16 or KEA_BF16. d a multiple of 8, at most 256; every pointer and stride
 *                a multiple of 16 bytes, strides not negative. out overlaps no input.
 *   kv_lengths   int32 [batch], NULL: tk for each.  q_starts: int32 [batch], NULL: len - tq (the last tokens).
 *   left, right  >= 0; 2^30 and above: without bound.  sinks >= 0.  tq, tk <= 2^30.  scale: finite.
 *   workspace    kea_window_attention_workspace bytes, 16-byte aligned (0: may be NULL): the unnormalised outputs, maxima and
 *                sums of parts of the keys where few queries meet many, written before they are read. */
int64_t kea_window_attention_workspace(int dtype, int64_t batch, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads,
                                       int64_t d, int64_t left, int64_t right, int64_t sinks);
int kea_window_attention(const kea_heads *q, const kea_heads *k, const kea_heads *v, const kea_heads *out, int dtype,
                         int64_t batch, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d, int64_t left,
                         int64_t right, int64_t sinks, float scale, const int32_t *kv_lengths_dev,
                         const int32_t *q_starts_dev, void *workspace_dev, int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* KEA_BLOCK_H */
