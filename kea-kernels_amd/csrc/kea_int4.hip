// int8 x int4 matrix product with group scales (include/kea_decode.h).
//
//   acc[m][n] = sum_g wscale[n][g] sum_{k in g} q[m][k] w[n][k]   on v_mfma_i32_16x16x64_i8, then scale, bias, SiLU, residual
//
// A lane's 16 bytes of the weight layout are its operand of two such instructions: word u of either is eight weights of its row
// in order, low nibbles first. (word << 4) & 0xF0F0F0F0 and word & 0xF0F0F0F0 are four int8 values of 16 times the weights each:
// three vector instructions for eight of them. The factor 16 leaves with the row's scale. The weights are the first operand, so
// lane 16 g + i ends up with columns 4 g .. 4 g + 3 of output row i.
//
// An integer sum is scaled after 128 k (groups of 128 and more), 64, or 32, for which the instruction runs twice, each time with
// the other half of q's k set to zero.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_epilogue.h"
#include "kea_internal.h"
#include "../../include/kea_decode.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
// Rows of outputs and of the residual start at any element: vectors of them, aligned to an element.
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4), aligned(2)));

struct Args {
    const int8_t *q;
    long long ldq;
    const uint32_t *words;
    const void *qs, *ws, *bias;
    void *y;
    long long ldy;
    const float *res;
    long long ldr;
    float factor;
    int m, n, k, blocks, groups, shift;  // blocks of 128 k; a block's first group is block * SCALES >> shift
    int qs_dtype, bias_dtype, y_dtype, flags;
};

// ---- operands and epilogue -----------------------------------------------------------------------------------------------------

// The int8 operand (16 times the weights) of half h of a lane's 16 bytes.
__device__ __forceinline__ v4i weights(v4i packed, int h) {
    const uint32_t a = (uint32_t)packed[2 * h], b = (uint32_t)packed[2 * h + 1];
    return v4i{(int)(a << 4 & 0xF0F0F0F0u), (int)(a & 0xF0F0F0F0u), (int)(b << 4 & 0xF0F0F0F0u), (int)(b & 0xF0F0F0F0u)};
}

template <typename ST>
__device__ __forceinline__ v4f scales4(const ST *p) {
    if constexpr (sizeof(ST) == 2) {
        const v4h v = *(const v4h *)p;
        return v4f{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    } else {
        return *(const v4f *)p;
    }
}

// acc += the scaled sums of one block of 128 k: w the lane's packed weights, q its operands of both halves, s the scales of its
// four columns, SCALES groups of them.
template <int SCALES>
__device__ __forceinline__ v4f block_product(v4i w, const v4i *q, const v4f *s, v4f acc, int g) {
    const v4i zero = {0, 0, 0, 0};
    v4i sum = zero;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const v4i wh = weights(w, h);
        if constexpr (SCALES == 4) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(wh, g / 2 == half ? q[h] : zero, zero, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf((float)sum[r], s[2 * h + half][r], acc[r]);
            }
        } else {
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(wh, q[h], SCALES == 2 ? zero : sum, 0, 0, 0);
            if (SCALES == 2 || h == 1)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf((float)sum[r], s[SCALES == 2 ? h : 0][r], acc[r]);
        }
    }
    return acc;
}

// Outputs [row][n0 .. n0 + 3] from their sums (16 times them); s the row's scale, b the columns' bias.
__device__ __forceinline__ void store4(const Args &p, int row, int n0, v4f acc, float s, const float *b) {
    const long long at = (long long)row * p.ldy + n0;
    const bool full = n0 + 3 < p.n;
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = kea::finish(acc[r] * 0.0625f, s, b[r], p.flags);
    if (p.res) {
        const float *res = p.res + (long long)row * p.ldr + n0;
        if (full) {
            const f32x4 x = *(const f32x4 *)res;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = x[r] + v[r] * p.factor;
        } else {
            for (int r = 0; r < 4; ++r)
                if (n0 + r < p.n) v[r] = res[r] + v[r] * p.factor;
        }
    }
    asm("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));  // rounded to FP32 before they are rounded to 16 bits
    if (p.y_dtype == KEA_F32) {
        float *y = (float *)p.y + at;
        if (full) *(f32x4 *)y = f32x4{v[0], v[1], v[2], v[3]};
        else
            for (int r = 0; r < 4; ++r)
                if (n0 + r < p.n) y[r] = v[r];
        return;
    }
    u16x4 h;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        h[r] = p.y_dtype == KEA_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[r]) : __builtin_bit_cast(uint16_t, (__bf16)v[r]);
    uint16_t *y = (uint16_t *)p.y + at;
    if (full) *(u16x4 *)y = h;
    else
        for (int r = 0; r < 4; ++r)
            if (n0 + r < p.n) y[r] = h[r];
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------

// A workgroup owns 16 RM rows of 16 columns; its NW waves share out the blocks of k, each loading its operands straight into
// registers, U blocks at once, and their sums meet in LDS, added in the waves' order.
template <int RM, int SCALES, typename ST, int NW, int U>
__global__ void __launch_bounds__(NW * 64) split_kernel(Args p, int tiles_n) {
    static_assert(RM <= NW, "a wave finishes one block at most");
    __shared__ v4f part[NW][RM][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
    const int m0 = blockIdx.x / tiles_n * (16 * RM), tile = blockIdx.x % tiles_n;
    const int from = (int)((long long)p.blocks * wave / NW), to = (int)((long long)p.blocks * (wave + 1) / NW);
    const int last = (p.k - 1) & ~15;  // the last 16 bytes of a row
    const v4i *const w = (const v4i *)p.words + ((long long)tile * p.blocks * 64 + lane);
    const ST *const ws = (const ST *)p.ws + ((long long)tile * p.groups * 16 + 4 * g);
    const int8_t *qr[RM];
#pragma unroll
    for (int a = 0; a < RM; ++a) qr[a] = p.q + (long long)min(m0 + 16 * a + i, p.m - 1) * p.ldq;
    v4f acc[RM];
#pragma unroll
    for (int a = 0; a < RM; ++a) acc[a] = v4f{0, 0, 0, 0};
    const v4i zero = {0, 0, 0, 0};
    for (int b0 = from; b0 < to; b0 += U) {
        v4i wf[U], qf[U][RM][2];
        v4f s[U][SCALES];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = min(b0 + u, to - 1);
            wf[u] = w[(long long)b * 64];
#pragma unroll
            for (int c = 0; c < SCALES; ++c) s[u][c] = scales4(ws + 16 * min((b * SCALES + c) >> p.shift, p.groups - 1));
#pragma unroll
            for (int a = 0; a < RM; ++a)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // (rows past the last have no loads; units past a row's end meet weights of zero)
                    qf[u][a][h] = m0 + 16 * a + i < p.m ? *(const v4i *)(qr[a] + min(128 * b + 64 * h + 16 * g, last)) : zero;
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b0 + u < to)
#pragma unroll
                for (int a = 0; a < RM; ++a) acc[a] = block_product<SCALES>(wf[u], qf[u][a], s[u], acc[a], g);
    }
#pragma unroll
    for (int a = 0; a < RM; ++a) part[wave][a][lane] = acc[a];
    __syncthreads();
    const int row = m0 + 16 * wave + i, col = 16 * tile + 4 * g;
    if (wave >= RM || row >= p.m || col >= p.n) return;
    v4f sum = part[0][wave][lane];
#pragma unroll
    for (int o = 1; o < NW; ++o) sum += part[o][wave][lane];
    float b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) b[r] = p.bias ? kea::load_scalar(p.bias, p.bias_dtype, min(col + r, p.n - 1)) : kea::kNoBias;
    store4(p, row, col, sum, kea::load_scalar(p.qs, p.qs_dtype, row), b);
}

// ---- host ----------------------------------------------------------------------------------------------------------------------

bool scale_type(int t) { return t == KEA_F32 || t == KEA_F16; }
bool aligned(const void *p, int dtype) { return (uintptr_t)p % (dtype == KEA_F32 ? 4 : 2) == 0; }

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_int4_gemm: ") + hipGetErrorString(e));
}

template <int RM, int SCALES, typename ST>
int run_split(const Args &a, hipStream_t stream) {
    constexpr int NW = 4;
    const int tn = (a.n + 15) / 16;
    const long long tiles = (long long)((a.m + 16 * RM - 1) / (16 * RM)) * tn;
    if (tiles > INT32_MAX / 2 || !kea::fits_dispatch(tiles, NW * 64)) return kea::fail(KEA_EINVAL, "kea_int4_gemm: too large for one launch");
    split_kernel<RM, SCALES, ST, NW, 4 / RM><<<dim3((unsigned)tiles), NW * 64, 0, stream>>>(a, tn);
    return launched();
}

template <int SCALES, typename ST>
int run(const Args &a, hipStream_t stream) {
    return a.m <= 16 ? run_split<1, SCALES, ST>(a, stream) : a.m <= 32 ? run_split<2, SCALES, ST>(a, stream) : run_split<4, SCALES, ST>(a, stream);
}

template <typename ST>
int run_group(const Args &a, int64_t group, hipStream_t stream) {
    return group == 32 ? run<4, ST>(a, stream) : group == 64 ? run<2, ST>(a, stream) : run<1, ST>(a, stream);
}

}  // namespace

extern "C" {

int kea_int4_gemm(const int8_t *q, int64_t ldq, const void *qs, int qs_dtype, const uint32_t *words, const void *wscale, int ws_dtype,
                  int64_t group, const void *bias, int bias_dtype, void *y, int y_dtype, int64_t ldy, const float *residual, int64_t ldr,
                  float factor, int64_t m, int64_t n, int64_t k, int flags, void *stream) {
    if (m < 0 || n < 1 || k < 1 || k > (1 << 20) || m > INT32_MAX - 4096 || n > INT32_MAX - 4096)
        return kea::fail(KEA_EINVAL, "kea_int4_gemm: sizes m >= 0, n >= 1, 1 <= k <= 2^20 below 2^31 are needed");
    if (group < 32 || group > (1 << 30) || (group & (group - 1))) return kea::fail(KEA_EINVAL, "kea_int4_gemm: a group is a power of two of 32 or more");
    if (ldq < k || ldy < n || (residual && ldr < n)) return kea::fail(KEA_EINVAL, "kea_int4_gemm: a leading dimension is below its row");
    if (y_dtype != KEA_F32 && y_dtype != KEA_F16 && y_dtype != KEA_BF16) return kea::fail(KEA_EINVAL, "kea_int4_gemm: y must be f32, f16 or bf16");
    if (flags & ~KEA_FLAG_SILU) return kea::fail(KEA_EINVAL, "kea_int4_gemm: the only flag is KEA_FLAG_SILU");
    if (!scale_type(qs_dtype) || !scale_type(ws_dtype) || (bias && !scale_type(bias_dtype)))
        return kea::fail(KEA_EINVAL, "kea_int4_gemm: scales and bias are f32 or f16");
    if (m == 0) return KEA_OK;
    if (!q || !words || !y || !qs || !wscale) return kea::fail(KEA_EINVAL, "kea_int4_gemm: a pointer is missing");
    if ((uintptr_t)q % 16 || (uintptr_t)words % 16 || (uintptr_t)wscale % 16 || ldq % 16)
        return kea::fail(KEA_EALIGN, "kea_int4_gemm: rows of q, the words and their scales start at multiples of 16 bytes");
    if (!aligned(y, y_dtype) || !aligned(qs, qs_dtype) || !aligned(bias, bias_dtype) || (uintptr_t)residual % 4)
        return kea::fail(KEA_EALIGN, "kea_int4_gemm: a pointer is not aligned to its element size");
    int shift = 0;
    while ((int64_t)128 << shift < group) ++shift;
    const Args a{q, ldq, words, qs, wscale, bias, y, ldy, residual, ldr, factor, (int)m, (int)n, (int)k, (int)((k + 127) / 128),
                 (int)((k + group - 1) / group), shift, qs_dtype, bias_dtype, y_dtype, flags};
    return ws_dtype == KEA_F16 ? run_group<_Float16>(a, group, (hipStream_t)stream) : run_group<float>(a, group, (hipStream_t)stream);
}

}  // extern "C"
