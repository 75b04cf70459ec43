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
 *   wscale   [ceil(n / 16)][ceil(k / group)][16], KEA_F32 or KEA_F16, 16-byte aligned; rows behind the matrix are zero. A sum is held
 *            as 16 acc: scales up to 2^113 / k in size keep it below FP32's largest number.
 *   group    a power of two, 32 or more.
 *   qs, bias KEA_F32 or KEA_F16 (bias may be NULL), aligned to their element size.
 *   residual NULL or FP32 [m][ldr]; y may be the residual itself (y_dtype KEA_F32, ldy == ldr) and overlaps no other operand.
 * 1 <= k <= 2^20. */
int kea_int4_gemm(const int8_t *q_dev, int64_t ldq, const void *qs_dev, int qs_dtype, const uint32_t *words_dev,
                  const void *wscale_dev, int ws_dtype, int64_t group, const void *bias_dev, int bias_dtype, void *y_dev,
                  int y_dtype, int64_t ldy, const float *residual_dev, int64_t ldr, float factor, int64_t m, int64_t n, int64_t k,
                  int flags, void *stream);

/* An int8 key or value cache in pages: row r (0 <= r < page_size) of head h of page i is d bytes at data_dev + i * page_stride +
 * h * head_stride + r * row_stride and one scale at scale_dev + i * scale_page_stride + h * scale_head_stride + r *
 * scale_row_stride; element e stands for data[e] * scale. data_dev and its strides are multiples of 16; no strides are negative;
 * no two rows share memory. */
typedef struct {
    int8_t *data_dev;
    float *scale_dev;
    int64_t page_stride, head_stride, row_stride, scale_page_stride, scale_head_stride, scale_row_stride;
} kea_pages;

/* Where the tokens of `batch` sequences stand. Position p of sequence b is row p % page_size of page table_dev[b * table_stride +
 * p / page_size]; an entry outside 0 .. pages-1 names no page. Sequence b holds len = kv_lengths_dev[b] positions, clamped to
 * 0 .. table_width * page_size, its new tokens among them. The new tokens of a call, `tokens` rows, are packed: sequence b has rows
 * q_offsets_dev[b] .. q_offsets_dev[b + 1] - 1 (ascending, held to 0 .. tokens), or, where q_offsets_dev is NULL, n = tokens / batch
 * rows from b * n on. The n rows of a sequence stand at its last positions: the i-th at len - n + i.
 * page_size: a power of two from 16 to 1024; table_width * page_size <= 2^30; tokens and batch below 2^30. Pointers are aligned to
 * four bytes. Everything is read on the device: lengths, offsets and table entries may change between replays. */
typedef struct {
    const int32_t *table_dev, *kv_lengths_dev, *q_offsets_dev;
    int64_t table_stride, table_width, batch, pages, page_size, tokens;
} kea_paging;

/* Writes new tokens' keys and values, [tokens][kv_heads][d] of `dtype` (KEA_F32, KEA_F16, KEA_BF16; batch_stride is not used), to
 * their places: a row x becomes s = max(max|x| / 127, 1e-30) and rint(x / s), as kea_quantize makes one part (s is held to the
 * largest number of which 127 s is finite); a row with an infinity or NaN becomes s = NaN and zeros. Tokens that stand at no position
 * (rows of no sequence, positions below 0, entries that name no page) are left out; nothing else is written. Tokens of one call that
 * stand at the same place are not ordered: what is written there is not defined. d: a multiple of 16 up to 256; k, v and their strides
 * multiples of 16 bytes, not negative. */
int kea_paged_write(const kea_heads *k, const kea_heads *v, int dtype, int64_t kv_heads, int64_t d, const kea_pages *k_pages,
                    const kea_pages *v_pages, const kea_paging *paging, void *stream);

/* Reads positions starts_dev[b] + i (starts_dev NULL: i), 0 <= i < length, of every sequence as values: k_dev, v_dev
 * [batch][length][kv_heads][d] of `dtype`, contiguous and 16-byte aligned: data * scale rounded to FP32, and from there to the 16-bit
 * types (a 16-bit result may lie half a step of FP32 more than half a step of its type from the product); zeros for positions
 * outside 0 .. len-1 and for entries that name no page. paging->tokens and q_offsets_dev are not used. */
int kea_paged_read(const kea_pages *k_pages, const kea_pages *v_pages, const kea_paging *paging, const int32_t *starts_dev,
                   int64_t length, int64_t kv_heads, int64_t d, void *k_dev, void *v_dev, int dtype, void *stream);

/* Attention of the new tokens q [tokens][heads][d] to the positions of their sequences (the new tokens' own keys and values are in
 * the cache): the token at position p sees position j iff p - left <= j <= p and the table names a page for j;
 *   out = sum_j softmax_j(scale * q . k_j) v_j over what it sees, zeros where it sees nothing or p is below 0.
 * Head h reads key head h / (heads / kv_heads). A position that a token does not see has no part in its output, whatever its scales
 * and codes are. Sums, maxima and scores are FP32; the weights exp(s - max) v_scale are rounded to FP16 (to two parts of it, 22
 * bits, with KEA_F32), small ones to multiples of 2^-30 of the row's largest such weight, and the elements of a row of q, with KEA_BF16
 * and KEA_F32, to 2^-28 of the row's largest (KEA_F32: 22 bits).
 *   dtype        of q and out: KEA_F32, KEA_F16 or KEA_BF16; pointers and strides multiples of 16 bytes, strides not negative
 *                (batch_stride is not used). out overlaps no input, and no two of its rows share memory.
 *   left         >= 0; 2^30 and above: without bound.  scale: finite.  Rows of a page less than 2^26 bytes apart.
 *   fill         0: rows of no sequence are left as they are; otherwise they become zeros.
 *   workspace    kea_paged_attention_workspace bytes (positions = table_width * page_size; offsets: whether q_offsets_dev is given),
 *                16-byte aligned (0: may be NULL): means, references and sums of parts of the keys, written before they are read. */
int64_t kea_paged_attention_workspace(int dtype, int64_t batch, int64_t tokens, int64_t positions, int64_t heads, int64_t kv_heads, int64_t d,
                                      int64_t left, int offsets);
int kea_paged_attention(const kea_heads *q, const kea_heads *out, int dtype, int64_t heads, int64_t kv_heads, int64_t d, const kea_pages *k_pages,
                        const kea_pages *v_pages, const kea_paging *paging, int64_t left, float scale, int fill, void *workspace_dev,
                        int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* KEA_DECODE_H */
