// The norms behind one block and before the next with the block's gate and residual scale (include/kea_block.h): one
// workgroup of 256 threads per row, the row held in LDS as FP32 between the passes.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_internal.h"
#include "kea_rowq.h"
#include "kea_wave.h"
#include "../../include/kea_block.h"

namespace {

struct Args {
    const void *x, *block, *gate;
    void *y, *z;
    int8_t *q;
    float *qs;
    long long ldx, ldb, ldg, ldy, ldz, ldq, gate_rows;
    kea_norm post, pre;
    float factor;
    int d, x_dtype, b_dtype, gate_act;
};

__device__ __forceinline__ float load(const void *p, int dtype, long long i) {
    if (dtype == KEA_F32) return ((const float *)p)[i];
    if (dtype == KEA_F16) return (float)((const _Float16 *)p)[i];
    return (float)((const __bf16 *)p)[i];
}
__device__ __forceinline__ void store(void *p, int dtype, long long i, float v) {
    asm("" : "+v"(v));  // rounded to FP32 before it is rounded to 16 bits
    if (dtype == KEA_F32) ((float *)p)[i] = v;
    else if (dtype == KEA_F16) ((_Float16 *)p)[i] = (_Float16)v;
    else ((__bf16 *)p)[i] = (__bf16)v;
}

template <bool MAX>
__device__ float reduce(float v, float *red) {
    v = MAX ? kea::wave_max(v) : kea::wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return MAX ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
}

// row[] -> norm(row[]); each thread touches its own elements only
__device__ void normalize(float *row, int d, const kea_norm &nm, float *red) {
    if (nm.kind == KEA_NORM_NONE) return;
    float mean = 0.0f, s = 0.0f;
    if (nm.kind == KEA_NORM_LAYER) {
        for (int i = threadIdx.x; i < d; i += 256) s += row[i];
        mean = reduce<false>(s, red) / (float)d;
    }
    s = 0.0f;
    for (int i = threadIdx.x; i < d; i += 256) s += (row[i] - mean) * (row[i] - mean);
    const float scale = 1.0f / sqrtf(reduce<false>(s, red) / (float)d + nm.eps);
    for (int i = threadIdx.x; i < d; i += 256) {
        float v = (row[i] - mean) * scale;
        if (nm.w_dev) v = v * load(nm.w_dev, nm.dtype, i);
        if (nm.b_dev) v = v + load(nm.b_dev, nm.dtype, i);
        row[i] = v;
    }
}

__global__ void __launch_bounds__(256) block_norm_kernel(Args a) {
    extern __shared__ float row[];
    __shared__ float red[4];
    const long long r = blockIdx.x;
    const int d = a.d, t = threadIdx.x;
    if (a.block) {
        for (int i = t; i < d; i += 256) row[i] = load(a.block, a.b_dtype, r * a.ldb + i);
        normalize(row, d, a.post, red);
        for (int i = t; i < d; i += 256) {
            float p = row[i];
            if (a.gate) {
                float g = load(a.gate, a.b_dtype, r / a.gate_rows * a.ldg + i);
                if (a.gate_act == KEA_GATE_SIGMOID) g = 1.0f / (1.0f + expf(-g));
                if (a.gate_act == KEA_GATE_TANH) g = tanhf(g);
                p = p * g;
            }
            const float v = load(a.x, a.x_dtype, r * a.ldx + i) + a.factor * p;
            row[i] = v;
            store(a.y, a.x_dtype, r * a.ldy + i, v);
        }
    } else {
        for (int i = t; i < d; i += 256) row[i] = load(a.x, a.x_dtype, r * a.ldx + i);
    }
    normalize(row, d, a.pre, red);
    if (a.z)
        for (int i = t; i < d; i += 256) store(a.z, a.b_dtype, r * a.ldz + i, row[i]);
    if (a.q) {
        float top = 0.0f;
        for (int i = t; i < d; i += 256) top = fmaxf(top, fabsf(row[i]));
        const float s = fmaxf(reduce<true>(top, red) / 127.0f, 1e-30f), inv = 1.0f / s;
        for (long long i = t; i < a.ldq; i += 256) {
            float v = i < d ? row[i] : 0.0f;
            a.q[r * a.ldq + i] = (int8_t)kea::quantize_code(v, s, inv);
        }
        if (t == 0) a.qs[r] = s;
    }
}

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
    if (!kea::fits_dispatch(m, 256)) return kea::fail(KEA_EINVAL, "kea_block_norm: too large for one launch");
    Args a{x, block, gate, y, z, q, qs, ldx, ldb, ldg, ldy, ldz, ldq, gate_rows, *post, *pre, factor, (int)d, x_dtype, block_dtype, gate_act};
    const size_t lds = (size_t)d * 4;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)block_norm_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return kea::fail((int)e, std::string("kea_block_norm: ") + hipGetErrorString(e));
    }
    block_norm_kernel<<<dim3((unsigned)m), 256, lds, (hipStream_t)stream>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_block_norm: ") + hipGetErrorString(e));
}
