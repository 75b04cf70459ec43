// int8 x int8 matrix product with a scale for each token and channel (include/kea_block.h).
//
//   acc[m][n] = sum_k q[m][k] w[n][k]   on v_mfma_i32_16x16x64_i8, then the epilogue of kea_epilogue.h
//
// One wave per 16 x 16 outputs. The weight rows are the instruction's first operand, so lane 16 g + i ends up with columns
// 4 g .. 4 g + 3 of output row i. Bytes of q from k on are masked to zero, so what w holds there does not matter.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_epilogue.h"
#include "kea_internal.h"
#include "../../include/kea_block.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

struct Args {
    const int8_t *q, *w;
    long long ldq, ldw;
    const void *qs, *ws, *bias;
    void *y;
    long long ldy;
    const float *res;
    long long ldr;
    float factor;
    int m, n, k;
    int qs_dtype, ws_dtype, bias_dtype, y_dtype, flags;
};

__device__ __forceinline__ void store_one(const Args &a, int row, int col, int acc) {
    const long long at = (long long)row * a.ldy + col;
    if (a.y_dtype == KEA_I32) {
        ((int32_t *)a.y)[at] = acc;
        return;
    }
    float r = (float)acc * kea::load_scalar(a.qs, a.qs_dtype, row);
    r = kea::finish(r, kea::load_scalar(a.ws, a.ws_dtype, col), a.bias != nullptr,
                    a.bias ? kea::load_scalar(a.bias, a.bias_dtype, col) : 0.0f, a.flags);
    if (a.res) r = a.res[(long long)row * a.ldr + col] + r * a.factor;
    asm("" : "+v"(r));  // rounded to FP32 before it is rounded to 16 bits
    if (a.y_dtype == KEA_F32) ((float *)a.y)[at] = r;
    else if (a.y_dtype == KEA_F16) ((_Float16 *)a.y)[at] = (_Float16)r;
    else ((__bf16 *)a.y)[at] = (__bf16)r;
}

// The 16 bytes of a row from k0 on, zero where k0 is past the row's end.
__device__ __forceinline__ v4i load16(const int8_t *row, int k0, int k) {
    if (k0 >= k) return v4i{0, 0, 0, 0};
    return *(const v4i *)(row + k0);
}
__device__ __forceinline__ v4i mask16(v4i v, int k0, int k) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int left = k - (k0 + 4 * d);
        if (left < 4) v[d] = left <= 0 ? 0 : v[d] & ((1 << (8 * left)) - 1);
    }
    return v;
}

__global__ void __launch_bounds__(256) int8_kernel(Args a) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const int tiles_n = (a.n + 15) / 16;
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int m0 = (int)(tile / tiles_n) * 16, n0 = (int)(tile % tiles_n) * 16;
    if (m0 >= a.m) return;
    const int8_t *qr = a.q + (long long)min(m0 + i, a.m - 1) * a.ldq;
    const int8_t *wr = a.w + (long long)min(n0 + i, a.n - 1) * a.ldw;
    v4i acc = {0, 0, 0, 0};
    for (int k0 = 16 * g; k0 - 16 * g < a.k; k0 += 64)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16(wr, k0, a.k), mask16(load16(qr, k0, a.k), k0, a.k), acc, 0, 0, 0);
    if (m0 + i < a.m)
        for (int r = 0; r < 4; ++r)
            if (n0 + 4 * g + r < a.n) store_one(a, m0 + i, n0 + 4 * g + r, acc[r]);
}

bool scale_type(int t) { return t == KEA_F32 || t == KEA_F16; }
bool aligned(const void *p, int dtype) { return (uintptr_t)p % (dtype == KEA_F32 || dtype == KEA_I32 ? 4 : 2) == 0; }

}  // namespace

extern "C" {

int64_t kea_int8_gemm_workspace(int64_t m, int64_t n, int64_t k) {
    if (m < 0 || n < 1 || k < 1) return kea::fail(KEA_EINVAL, "kea_int8_gemm_workspace: m >= 0, n >= 1 and k >= 1 are needed");
    return 0;
}

int kea_int8_gemm(const int8_t *q, int64_t ldq, const void *qs, int qs_dtype, const int8_t *w, int64_t ldw, const void *wscale,
                  int ws_dtype, const void *bias, int bias_dtype, void *y, int y_dtype, int64_t ldy, const float *residual,
                  int64_t ldr, float factor, int64_t m, int64_t n, int64_t k, int flags, void *workspace,
                  int64_t workspace_bytes, void *stream) {
    if (m < 0 || n < 1 || k < 1 || k > 131071 || m > INT32_MAX - 4096 || n > INT32_MAX - 4096)
        return kea::fail(KEA_EINVAL, "kea_int8_gemm: sizes m >= 0, n >= 1, 1 <= k <= 131071 below 2^31 are needed");
    if (ldq < k || ldw < k || ldy < n || (residual && ldr < n))
        return kea::fail(KEA_EINVAL, "kea_int8_gemm: a leading dimension is below its row");
    if (y_dtype != KEA_F32 && y_dtype != KEA_F16 && y_dtype != KEA_BF16 && y_dtype != KEA_I32)
        return kea::fail(KEA_EINVAL, "kea_int8_gemm: y must be f32, f16, bf16 or int32");
    if (flags & ~KEA_FLAG_SILU) return kea::fail(KEA_EINVAL, "kea_int8_gemm: the only flag is KEA_FLAG_SILU");
    if (y_dtype == KEA_I32 ? (bias || residual || flags) : (!scale_type(qs_dtype) || !scale_type(ws_dtype) || (bias && !scale_type(bias_dtype))))
        return kea::fail(KEA_EINVAL, "kea_int8_gemm: scales and bias are f32 or f16; int32 sums take no bias, residual or flags");
    if (m == 0) return KEA_OK;
    if (!q || !w || !y || (y_dtype != KEA_I32 && (!qs || !wscale))) return kea::fail(KEA_EINVAL, "kea_int8_gemm: a pointer is missing");
    if ((uintptr_t)q % 16 || (uintptr_t)w % 16 || ldq % 16 || ldw % 16)
        return kea::fail(KEA_EALIGN, "kea_int8_gemm: rows of q and w start at multiples of 16 bytes");
    if (!aligned(y, y_dtype) || !aligned(qs, qs_dtype) || !aligned(wscale, ws_dtype) || !aligned(bias, bias_dtype) || (uintptr_t)residual % 4)
        return kea::fail(KEA_EALIGN, "kea_int8_gemm: a pointer is not aligned to its element size");
    Args a{q, w, ldq, ldw, qs, wscale, bias, y, ldy, residual, ldr, factor, (int)m, (int)n, (int)k,
           qs_dtype, ws_dtype, bias_dtype, y_dtype, flags};
    const int64_t tiles = (m + 15) / 16 * ((n + 15) / 16);
    if (!kea::fits_dispatch((tiles + 3) / 4, 256)) return kea::fail(KEA_EINVAL, "kea_int8_gemm: too large for one launch");
    int8_kernel<<<dim3((unsigned)((tiles + 3) / 4)), 256, 0, (hipStream_t)stream>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_int8_gemm: ") + hipGetErrorString(e));
}

}  // extern "C"
