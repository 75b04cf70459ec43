// The norms behind one block and before the next with the block's gate and residual scale (include/kea_block.h): the host
// side. The row kernels are in kea_norm_inst.h.
#include <hip/hip_runtime.h>

#include <string>

#include "kea_norm.h"

namespace {

bool value_type(int t) { return t == KEA_F32 || t == KEA_F16 || t == KEA_BF16; }
bool aligned(const void *p, int dtype) { return (uintptr_t)p % (dtype == KEA_F32 ? 4 : 2) == 0; }
bool norm_ok(const kea_norm &n) {
    return n.kind == KEA_NORM_NONE || ((n.kind == KEA_NORM_LAYER || n.kind == KEA_NORM_RMS) && value_type(n.dtype) &&
                                       aligned(n.w_dev, n.dtype) && aligned(n.b_dev, n.dtype));
}

}  // namespace

extern "C" int kea_block_norm(const void *x, int x_dtype, int64_t ldx, const void *block, int block_dtype, int64_t ldb, int64_t m,
                              int64_t d, const kea_norm *post, const void *gate, int64_t ldg, int64_t gate_rows, int gate_act,
                              float factor, void *y, int64_t ldy, const kea_norm *pre, void *z, int64_t ldz, int8_t *q,
                              int64_t ldq, float *qs, void *stream) {
    if (m < 0 || d < 1 || d > 32768) return kea::fail(KEA_EINVAL, "kea_block_norm: m >= 0 and 1 <= d <= 32768 are needed");
    if (!value_type(x_dtype) || !value_type(block_dtype)) return kea::fail(KEA_EINVAL, "kea_block_norm: x and block are f32, f16 or bf16");
    if (!post || !pre || !norm_ok(*post) || !norm_ok(*pre))
        return kea::fail(KEA_EINVAL, "kea_block_norm: a norm's kind is 0, 1 or 2 and its parameters f32, f16 or bf16, aligned to their size");
    if (gate_act < 0 || gate_act > KEA_GATE_TANH || gate_rows < 1) return kea::fail(KEA_EINVAL, "kea_block_norm: gate_act is 0, 1 or 2 and gate_rows >= 1");
    if (ldx < d || (block && (ldb < d || ldy < d)) || (gate && ldg < d) || (z && ldz < d) || (q && ldq < d))
        return kea::fail(KEA_EINVAL, "kea_block_norm: a leading dimension is below its row");
    if ((!block && (gate || y || post->kind != KEA_NORM_NONE)) || (z && (pre->kind == KEA_NORM_NONE || q)) || (q && !qs))
        return kea::fail(KEA_EINVAL, "kea_block_norm: no gate, y or post without a block; z needs a norm, q its scales, and one excludes the other");
    if (m == 0) return KEA_OK;
    if (!x || (block && !y) || (!block && !z && !q)) return kea::fail(KEA_EINVAL, "kea_block_norm: a pointer is missing");
    if (!aligned(x, x_dtype) || !aligned(block, block_dtype) || !aligned(gate, block_dtype) || !aligned(y, x_dtype) || !aligned(z, block_dtype) || (uintptr_t)qs % 4)
        return kea::fail(KEA_EALIGN, "kea_block_norm: a pointer is not aligned to its element size");
    const unsigned threads = d <= 512 ? 64 : d <= 1024 ? 128 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024;  // of a row
    if (m > UINT32_MAX || !kea::fits_dispatch(m + 3, threads)) return kea::fail(KEA_EINVAL, "kea_block_norm: too large for one launch");
    const kea::NormArgs a{x, block, gate, y, z, q, qs, m, ldx, ldb, ldg, ldy, ldz, ldq, gate_rows, *post, *pre, factor, (int)d, block_dtype, gate_act};
    if (x_dtype == KEA_F32) kea::norm_rows<float>(a, stream);
    else if (x_dtype == KEA_F16) kea::norm_rows<_Float16>(a, stream);
    else kea::norm_rows<__bf16>(a, stream);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_block_norm: ") + hipGetErrorString(e));
}
