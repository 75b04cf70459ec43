// kea_block_norm's launch parameters, shared by its host side and the row kernels of each stream type.
#pragma once

#include "kea_internal.h"
#include "../../include/kea_block.h"

namespace kea {

struct NormArgs {
    const void *x, *block, *gate;
    void *y, *z;
    int8_t *q;
    float *qs;
    long long m, ldx, ldb, ldg, ldy, ldz, ldq, gate_rows;
    kea_norm post, pre;
    float factor;
    int d, b_dtype, gate_act;
};

// Enqueues the rows for streams (x and y) of type T: float, _Float16 or __bf16 (kea_norm_f32.hip and its like).
template <typename T>
void norm_rows(const NormArgs &a, void *stream);
template <>
void norm_rows<float>(const NormArgs &a, void *stream);
template <>
void norm_rows<_Float16>(const NormArgs &a, void *stream);
template <>
void norm_rows<__bf16>(const NormArgs &a, void *stream);

}  // namespace kea
