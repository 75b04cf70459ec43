// Where the tokens of sequences stand in an int8 cache in pages (include/kea_decode.h): the arguments and lookups that the kernels
// which write, read and attend to it share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_internal.h"
#include "../../include/kea_decode.h"

namespace kea {

struct Paging {
    const int32_t *table, *lengths, *offsets;
    long long table_stride;
    int batch, width, pages, shift, tokens, each;  // a page holds 2^shift positions; each: tokens of a sequence without offsets

    // The positions that sequence b holds.
    __device__ __forceinline__ int length(int b) const { return min(max(lengths[b], 0), width << shift); }
    // The first row of sequence b and the row behind its last.
    __device__ __forceinline__ int2 rows(int b) const {
        if (!offsets) return make_int2(b * each, b * each + each);
        const int from = min(max(offsets[b], 0), tokens);
        return make_int2(from, min(max(offsets[b + 1], from), tokens));
    }
    // The sequence that has row t, -1 for none: as many offsets behind the first as are not above t, found by halving.
    __device__ __forceinline__ int sequence(int t) const {
        if (!offsets) return t / each;
        int b = 0, n = batch;
        while (n > 0) {
            const int half = n / 2;
            const bool past = offsets[b + half + 1] <= t;
            b = past ? b + half + 1 : b;
            n = past ? n - half - 1 : half;
        }
        return b < batch && t >= offsets[b] && t < offsets[b + 1] ? b : -1;
    }
    // The page of position p (0 <= p < width << shift) of sequence b, -1 for none.
    __device__ __forceinline__ int page(int b, int p) const {
        const int i = table[(long long)b * table_stride + (p >> shift)];
        return (unsigned)i < (unsigned)pages ? i : -1;
    }
};

inline bool pages_ok(const kea_pages *p) {
    return p && p->page_stride >= 0 && p->head_stride >= 0 && p->row_stride >= 0 && p->scale_page_stride >= 0 && p->scale_head_stride >= 0 &&
           p->scale_row_stride >= 0 && (uintptr_t)p->data_dev % 16 == 0 && p->page_stride % 16 == 0 && p->head_stride % 16 == 0 &&
           p->row_stride % 16 == 0 && (uintptr_t)p->scale_dev % 4 == 0;
}

// KEA_OK and the kernels' form of the arguments, or the error.
inline int check_paging(const char *what, const kea_pages *k, const kea_pages *v, const kea_paging *g, int64_t kv_heads, int64_t d, Paging *out) {
    const std::string name(what);
    if (!g || g->batch < 0 || g->batch >= (1 << 30) || g->tokens < 0 || g->tokens >= (1 << 30) || g->pages < 0 || g->pages > INT32_MAX || g->table_width < 0 || g->table_stride < 0)
        return fail(KEA_EINVAL, name + ": batch, tokens, pages and the table's width are >= 0 and below 2^30");
    if (g->page_size < 16 || g->page_size > 1024 || (g->page_size & (g->page_size - 1))) return fail(KEA_EINVAL, name + ": a page holds a power of two of 16 to 1024 positions");
    if (g->table_width > (1 << 30) / g->page_size) return fail(KEA_EINVAL, name + ": more than 2^30 positions");
    if (kv_heads < 1 || kv_heads > 65535 || d < 16 || d > 256 || d % 16) return fail(KEA_EINVAL, name + ": 1 to 65535 heads of a multiple of 16, 16 to 256, elements");
    if (!g->q_offsets_dev && (g->batch > 0 ? g->tokens % g->batch : g->tokens)) return fail(KEA_EINVAL, name + ": without offsets every sequence has as many tokens");
    if (!pages_ok(k) || !pages_ok(v)) return fail(KEA_EALIGN, name + ": pages and their strides are multiples of 16 bytes, strides not negative");
    if ((uintptr_t)g->table_dev % 4 || (uintptr_t)g->kv_lengths_dev % 4 || (uintptr_t)g->q_offsets_dev % 4)
        return fail(KEA_EALIGN, name + ": the table, lengths and offsets are aligned to four bytes");
    if (g->batch > 0 && (!g->kv_lengths_dev || (g->table_width > 0 && !g->table_dev) || (g->pages > 0 && (!k->data_dev || !v->data_dev || !k->scale_dev || !v->scale_dev))))
        return fail(KEA_EINVAL, name + ": a pointer is missing");
    int shift = 0;
    while ((1 << shift) < g->page_size) ++shift;
    // (no pages: no positions)
    *out = Paging{g->table_dev, g->kv_lengths_dev, g->q_offsets_dev, g->table_stride, (int)g->batch, g->pages > 0 ? (int)g->table_width : 0, (int)g->pages, shift,
                  (int)g->tokens, g->batch > 0 ? (int)(g->tokens / g->batch) : 0};
    return KEA_OK;
}

}  // namespace kea
