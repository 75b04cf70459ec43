/*
 * kea_decode.h - the operators of a decoder's layer with 4-bit weights and an 8-bit cache in libkea_hip.so (MI355X / gfx950): the
 * int8 x int4 matrix product with group scales, an int8 key/value cache in pages, and attention over it.
 *
 * Conventions as in kea_lowbit.h: device pointers, int64 sizes and strides (in elements), a hipStream_t as void*,
 * KEA_OK / negative KEA_E* (nothing launched) / positive hipError_t, message in kea_last_error(). No allocation, no
 * host synchronisation: every entry point can be captured into a HIP graph. The reference has no counterpart of these.
 */
#ifndef KEA_DECODE_H
#define KEA_DECODE_H

#include <stdint.h>

#include "kea_block.h"

#ifdef __cplusplus
extern "C" {
#endif

/* int8 x int4 matrix product with a scale for each row of q (token) and each `group` weights of a row of w:
 *   acc[m][n] = sum_g wscale[n][g] * S_g,   S_g = sum over the k of group g of q[m*ldq + k] * w[n][k]
 *   r = acc * qs[m];  r = bias ? r + bias[n] : r;  r = r / (1 + exp(-r)) with KEA_FLAG_SILU
 *   y[m*ldy + n] = RN(residual ? residual[m*ldr + n] + r * factor : r)     in y_dtype (KEA_F32, KEA_F16, KEA_BF16)
 * Integer sums are exact (of a group, or of 128 k where a group is longer), their scaled sum and all else is FP32.
 *   q, qs    as kea_quantize writes them with one part: rows of 16-byte aligned starts (pointer and ldq multiples of 16,
 *            ldq >= k); bytes at k and behind take no part, and none from the last row's k, rounded up to 16, on is read.
 *   words    w as two's complement nibbles in tiles of 16 rows and 128 k, 1024 bytes each, [ceil(n / 16)][ceil(k / 128)]: 16 bytes
 *            for each lane 16 j + i (i: the row in the tile): byte 8 h + 4 u + b holds in its low nibble k = 64 h + 16 j + 8 u + b
 *            and in its high nibble the k 4 further on. Rows and k behind the matrix are zero. 16-byte aligned.
 *   wscale   [ceil(n / 16)][ceil(k / group)][16], KEA_F32 or KEA_F16, 16-byte aligned; rows behind the matrix are zero.
 *   group    a power of two, 32 or more.
 *   qs, bias KEA_F32 or KEA_F16 (bias may be NULL), aligned to their element size.
 *   residual NULL or FP32 [m][ldr]; y may be the residual itself (y_dtype KEA_F32, ldy == ldr) and overlaps no other operand.
 * 1 <= k <= 2^20. */
int kea_int4_gemm(const int8_t *q_dev, int64_t ldq, const void *qs_dev, int qs_dtype, const uint32_t *words_dev,
                  const void *wscale_dev, int ws_dtype, int64_t group, const void *bias_dev, int bias_dtype, void *y_dev,
                  int y_dtype, int64_t ldy, const float *residual_dev, int64_t ldr, float factor, int64_t m, int64_t n, int64_t k,
                  int flags, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* KEA_DECODE_H */
