// The row kernel of kea_block_norm and its launch for one stream type; each kea_norm_*.hip defines KEA_NORM_STREAM.
//
// y = x + factor * act(gate) * post(block), z = pre(y). A row stays in registers from its loads to its stores: W waves hold
// it as N vectors of eight elements a thread, so each input is read once and each output written once. Memory bounds it:
// 16000 rows of 4096, BF16, with a tanh gate and two RMS norms, take 103 us, 5.1 TB/s, a large copy's rate; one such row takes
// 3.5 us, mostly the launch and the loads' latency. The sums of a norm are a wave's reduction and, where W > 1, one exchange
// of wave totals through LDS. The row's loads are issued together; the norms' parameters, which every row reads, come from
// the caches when they are used. The variance is the mean of the squared differences from the mean, a second reduction
// over registers.
//
// Vectors are accessed at any alignment of their elements. Where d is no multiple of 8, the last vector is moved back to end
// with the row: the elements that it shares with its neighbour are left out of the sums and not stored.
#include <hip/hip_runtime.h>

#include "kea_norm.h"
#include "kea_rowq.h"
#include "kea_wave.h"

namespace {

using kea::NormArgs;

template <typename T>
struct Eight {  // as they lie in memory
    typedef T v __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(1)));

// Elements e .. e + 7 of a row as FP32. TINY: rows of d < 8 elements, zeros behind them.
template <bool TINY, typename T>
__device__ __forceinline__ typename Eight<T>::v load8(const T *row, int e, int d) {
    if constexpr (!TINY) return *(const typename Eight<T>::v *)(row + e);
    typename Eight<T>::v r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = e + j < d ? row[min(e + j, d - 1)] : (T)0.0f;
    return r;
}
template <bool TINY, typename T>
__device__ __forceinline__ void floats8(const T *row, int e, int d, float (&v)[8]) {
    const auto r = load8<TINY>(row, e, d);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
}
template <bool TINY>
__device__ __forceinline__ void parameters8(const void *p, int dtype, int e, int d, float (&v)[8]) {
    if (dtype == KEA_F32) floats8<TINY>((const float *)p, e, d, v);
    else if (dtype == KEA_F16) floats8<TINY>((const _Float16 *)p, e, d, v);
    else floats8<TINY>((const __bf16 *)p, e, d, v);
}
// Elements lo .. hi - 1 of the eight at e.
template <typename T>
__device__ __forceinline__ void store8(T *row, int e, int lo, int hi, const float (&v)[8]) {
    typename Eight<T>::v r;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float x = v[j];
        asm("" : "+v"(x));  // rounded to FP32 before it is rounded to 16 bits
        r[j] = (T)x;
    }
    if (lo == 0 && hi == 8) {
        *(typename Eight<T>::v *)(row + e) = r;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= lo && j < hi) row[e + j] = r[j];
    }
}

// The sum (maximum) over a row's W waves; `slot`: a place of its own in LDS for each reduction of the kernel.
template <int W, bool MAX>
__device__ __forceinline__ float reduce(float v, float (*red)[W], int slot) {
    v = MAX ? kea::wave_max(v) : kea::wave_sum(v);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) red[slot][threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[slot][0];
#pragma unroll
        for (int w = 1; w < W; ++w) v = MAX ? fmaxf(v, red[slot][w]) : v + red[slot][w];
    }
    return v;
}

template <typename XT, typename BT, int N, int W, bool TINY>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) block_norm_kernel(NormArgs a) {
    __shared__ float red[5][W];
    const int d = a.d, t = W == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
    const long long r = W == 1 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (W == 1 && r >= a.m) return;
    // vector i of this thread: elements at[i] + lo[i] .. at[i] + hi - 1 of the row (none where lo is 8)
    int at[N], lo[N];
    const int hi = TINY ? d : 8;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = (t + i * 64 * W) * 8;
        at[i] = TINY ? 0 : min(e, d - 8);
        lo[i] = TINY ? (t ? 8 : 0) : min(e - at[i], 8);
    }
    // elements that belong to the neighbour, or to none, are zero
    auto clear = [&](float (&v)[N][8]) {
        if (!TINY && N * W * 512 == d) return;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < lo[i] || j >= hi) v[i][j] = 0.0f;
    };
    auto normalize = [&](float (&v)[N][8], const kea_norm &nm, int slot) {
        if (nm.kind == KEA_NORM_NONE) return;
        const float inv = 1.0f / (float)d;
        if (nm.kind == KEA_NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) s += v[i][j];
            const float mean = reduce<W, false>(s, red, slot) * inv;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] - mean;
            clear(v);
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[i][j] * v[i][j];
        const float scale = 1.0f / sqrtf(reduce<W, false>(s, red, slot + 1) * inv + nm.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * scale;
            float p[8];
            if (nm.w_dev) {
                parameters8<TINY>(nm.w_dev, nm.dtype, at[i], d, p);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * p[j];
            }
            if (nm.b_dev) {
                parameters8<TINY>(nm.b_dev, nm.dtype, at[i], d, p);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] + p[j];
            }
        }
    };

    const XT *const xr = (const XT *)a.x + r * a.ldx;
    float v[N][8];
    if (a.block) {
        typename Eight<BT>::v o[N], g[N];
        typename Eight<XT>::v x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = load8<TINY>((const BT *)a.block + r * a.ldb, at[i], d);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = load8<TINY>(xr, at[i], d);
        if (a.gate)
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = load8<TINY>((const BT *)a.gate + r / a.gate_rows * a.ldg, at[i], d);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = (float)o[i][j];
        clear(v);
        normalize(v, a.post, 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (a.gate) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = (float)g[i][j];
                if (a.gate_act == KEA_GATE_SIGMOID)
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(f[j] * -1.4426950408889634f));
                if (a.gate_act == KEA_GATE_TANH)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        // 1 - 2 / (1 + e^(2 g)), to 2^-22 of 1; below 1/4, where that is not enough of g, its series to g^9, whose
                        // next term is 2^-26 of g (16000 rows of 4096: 103 us, 99 without the series)
                        const float u = f[j] * f[j];
                        const float inner = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(62.0f / 2835, u, -17.0f / 315), u, 2.0f / 15), u, -1.0f / 3);
                        const float series = __builtin_fmaf(f[j] * u, inner, f[j]);
                        const float whole = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(f[j] * 2.8853900817779268f)), 1.0f);
                        f[j] = fabsf(f[j]) < 0.25f ? series : whole;
                    }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * f[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = (float)x[i][j] + a.factor * v[i][j];
            if (lo[i] < 8) store8((XT *)a.y + r * a.ldy, at[i], lo[i], hi, v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) floats8<TINY>(xr, at[i], d, v[i]);
    }
    if (!a.z && !a.q) return;
    clear(v);
    normalize(v, a.pre, 2);
    if (a.z) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lo[i] < 8) store8((BT *)a.z + r * a.ldz, at[i], lo[i], hi, v[i]);
    }
    if (a.q) {
        clear(v);
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[i][j]));
        const float s = fmaxf(reduce<W, true>(top, red, 4) / 127.0f, 1e-30f), inv = 1.0f / s;
        int8_t *const qr = a.q + r * a.ldq;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (lo[i] == 8) continue;
            u32x2 w = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j / 4] |= kea::quantize_code(v[i][j], s, inv) << (j % 4 * 8);
            if (lo[i] == 0 && hi == 8) {
                *(u32x2 *)(qr + at[i]) = w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j >= lo[i] && j < hi) qr[at[i] + j] = (int8_t)(w[j / 4] >> (j % 4 * 8));
            }
        }
        for (long long e = d + t; e < a.ldq; e += 64 * W) qr[e] = 0;
        if (t == 0) a.qs[r] = s;
    }
}

template <typename XT, typename BT, int N, int W, bool TINY = false>
void launch(const NormArgs &a, hipStream_t stream) {
    if (W == 1) block_norm_kernel<XT, BT, N, W, TINY><<<dim3((unsigned)((a.m + 3) / 4)), 256, 0, stream>>>(a);
    else block_norm_kernel<XT, BT, N, W, TINY><<<dim3((unsigned)a.m), 64 * W, 0, stream>>>(a);
}

// As many waves as hold the row in one vector a thread, up to sixteen: one row of 4096 takes 3.8 us so, 4.8 in four waves of two
// vectors and 6.6 in two of four; 16000 of them (FP32 streams, FP16 blocks) 152, 163 and 161. Rows of 8192 are alike (4.7
// against 7.0 in four waves of four, 16000 of them 289 and 298, but 1000 of them 22 and 20).
template <typename XT, typename BT>
void rows(const NormArgs &a, hipStream_t s) {
    if (a.d < 8) launch<XT, BT, 1, 1, true>(a, s);
    else if (a.d <= 512) launch<XT, BT, 1, 1>(a, s);
    else if (a.d <= 1024) launch<XT, BT, 1, 2>(a, s);
    else if (a.d <= 2048) launch<XT, BT, 1, 4>(a, s);
    else if (a.d <= 4096) launch<XT, BT, 1, 8>(a, s);
    else if (a.d <= 8192) launch<XT, BT, 1, 16>(a, s);
    else if (a.d <= 16384) launch<XT, BT, 2, 16>(a, s);
    else launch<XT, BT, 4, 16>(a, s);
}

}  // namespace

namespace kea {

template <>
void norm_rows<KEA_NORM_STREAM>(const NormArgs &a, void *stream) {
    if (a.b_dtype == KEA_F32) rows<KEA_NORM_STREAM, float>(a, (hipStream_t)stream);
    else if (a.b_dtype == KEA_F16) rows<KEA_NORM_STREAM, _Float16>(a, (hipStream_t)stream);
    else rows<KEA_NORM_STREAM, __bf16>(a, (hipStream_t)stream);
}

}  // namespace kea
