// Writing tokens' keys and values to an int8 cache in pages, and reading them back (include/kea_decode.h).
//
//   s = max(max|x| / 127, 1e-30), held to where 127 s is finite, c = rint(x / s) for each row x of d elements;   x' = c s
//
// Either moves bytes and little else: L = 4, 8 or 16 lanes of sixteen elements take a row, one head of a token or position; keys and
// values are two halves of the grid. Memory bounds both (16000 F16 tokens, 8 heads of 128: 99 MB written in 24.6 us, 4.0 TB/s, read back
// in 21.1, 4.7; eight sequences of up to 4000, 5.8 TB/s; a large copy's two directions together make 5.3), for few tokens a launch and
// three loads in line (length, page, row): 3.8 us for 16. A wave for each token or position, its heads in line, took 76 us for
// both where these two launches take 50 (calls in a row).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_internal.h"
#include "kea_pages.h"
#include "kea_rowq.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint16_t v8u __attribute__((ext_vector_type(8)));

constexpr float kMostScale = 0x1.0204060000000p+121f;  // the largest s of which 127 s is a finite number
constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T *p, float *v) {
    if constexpr (sizeof(T) == 4) {
        const v4f a = *(const v4f *)p, b = *(const v4f *)(p + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < 4 ? a[e & 3] : b[e & 3];
    } else {
        const v8u a = *(const v8u *)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t bits = a[e];
            v[e] = (float)__builtin_bit_cast(T, bits);
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float *v) {
    if constexpr (sizeof(T) == 4) {
        *(v4f *)p = v4f{v[0], v[1], v[2], v[3]};
        *(v4f *)(p + 4) = v4f{v[4], v[5], v[6], v[7]};
    } else {
        v8u a;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = __builtin_bit_cast(uint16_t, (T)v[e]);
        *(v8u *)p = a;
    }
}

// The largest of L neighbouring lanes' numbers, in all of them.
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    auto dpp = [](uint32_t v, auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, false); };
    v = max(v, dpp(v, std::integral_constant<int, 0xB1>{}));   // l ^ 1
    v = max(v, dpp(v, std::integral_constant<int, 0x4E>{}));   // l ^ 2
    if constexpr (L >= 8) v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));   // the other four of eight
    if constexpr (L >= 16) v = max(v, dpp(v, std::integral_constant<int, 0x140>{}));  // the other eight of 16
    return v;
}

struct WriteArgs {
    kea_heads k, v;
    kea_pages kp, vp;
    kea::Paging at;
    int kv_heads, d;
};

template <typename T, int L>
__global__ void __launch_bounds__(kThreads) write_kernel(WriteArgs a) {
    const long long r = (long long)blockIdx.x * (kThreads / L) + threadIdx.x / L;
    if (r >= (long long)a.at.tokens * a.kv_heads) return;
    const int t = (int)(r / a.kv_heads), h = (int)(r - (long long)t * a.kv_heads), at = threadIdx.x % L * 16;
    const kea_heads &from = blockIdx.y ? a.v : a.k;
    const kea_pages &to = blockIdx.y ? a.vp : a.kp;
    float x[16];
    uint32_t most = 0;  // (as whole numbers the sizes keep their order, with infinities and NaN on top)
    const T *const src = (const T *)from.data_dev + (long long)t * from.t_stride + (long long)h * from.head_stride + at;
    if (at < a.d) {
        load8(src, x);
        load8(src + 8, x + 8);
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.0f;
    }
    // where the token stands, while its elements are on their way
    const int b = a.at.sequence(t);
    int p = -1, page = -1;
    if (b >= 0) {
        p = a.at.length(b) - a.at.rows(b).y + t;  // len - n + i
        if (p >= 0) page = a.at.page(b, p);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) most = max(most, __builtin_bit_cast(uint32_t, x[e]) & 0x7FFFFFFFu);
    most = lanes_max<L>(most);
    const bool number = most < 0x7F800000u;
    const float s = number ? fminf(fmaxf(__builtin_bit_cast(float, most) / 127.0f, 1e-30f), kMostScale) : __builtin_nanf(""), inv = 1.0f / s;
    if (page < 0 || at >= a.d) return;
    v4u w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t code[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) code[e] = number ? kea::quantize_code(x[4 * i + e], s, inv) : 0u;
        w[i] = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
    }
    const int row = p & ((1 << a.at.shift) - 1);
    *(v4u *)(to.data_dev + page * to.page_stride + h * to.head_stride + row * to.row_stride + at) = w;
    if (at == 0) to.scale_dev[page * to.scale_page_stride + h * to.scale_head_stride + row * to.scale_row_stride] = s;
}

struct ReadArgs {
    kea_pages kp, vp;
    kea::Paging at;
    const int32_t *starts;
    void *k, *v;
    int kv_heads, d, length;
};

template <typename T, int L>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs a) {
    // (a grid has at most 65535 rows: more sequences lie behind each other in z, keys and values in turn)
    const int r = blockIdx.x * (kThreads / L) + threadIdx.x / L, b = blockIdx.z / 2 * gridDim.y + blockIdx.y, at = threadIdx.x % L * 16;
    const bool values = blockIdx.z % 2;
    if (b >= a.at.batch || r >= a.length * a.kv_heads || at >= a.d) return;
    const int i = r / a.kv_heads, h = r - i * a.kv_heads;
    const kea_pages &from = values ? a.vp : a.kp;
    const long long p = (a.starts ? (long long)a.starts[b] : 0) + i;
    const int page = p >= 0 && p < a.at.length(b) ? a.at.page(b, (int)p) : -1;
    v4u c = {0, 0, 0, 0};
    float s = 0.0f;
    if (page >= 0) {
        const int row = (int)p & ((1 << a.at.shift) - 1);
        c = *(const v4u *)(from.data_dev + page * from.page_stride + h * from.head_stride + row * from.row_stride + at);
        s = from.scale_dev[page * from.scale_page_stride + h * from.scale_head_stride + row * from.scale_row_stride];
    }
    T *const to = (T *)(values ? a.v : a.k) + ((long long)b * a.length * a.kv_heads + r) * a.d + at;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)(c[2 * half + e / 4] >> (8 * (e % 4))) * s;
        store8(to + 8 * half, x);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string(what) + ": " + hipGetErrorString(e));
}

bool type_ok(int t) { return t == KEA_F32 || t == KEA_F16 || t == KEA_BF16; }

bool rows_ok(const kea_heads *t, int64_t unit) {
    return t && t->t_stride >= 0 && t->head_stride >= 0 && (uintptr_t)t->data_dev % 16 == 0 && t->t_stride % unit == 0 && t->head_stride % unit == 0;
}

template <typename T>
int run_write(const WriteArgs &a, hipStream_t stream) {
    const int lanes = a.d <= 64 ? 4 : a.d <= 128 ? 8 : 16;
    const int64_t rows = (int64_t)a.at.tokens * a.kv_heads, blocks = (rows + kThreads / lanes - 1) / (kThreads / lanes);
    if (!kea::fits_dispatch(blocks, kThreads)) return kea::fail(KEA_EINVAL, "kea_paged_write: too large for one launch");
    const dim3 grid((unsigned)blocks, 2);
    if (lanes == 4) write_kernel<T, 4><<<grid, kThreads, 0, stream>>>(a);
    else if (lanes == 8) write_kernel<T, 8><<<grid, kThreads, 0, stream>>>(a);
    else write_kernel<T, 16><<<grid, kThreads, 0, stream>>>(a);
    return launched("kea_paged_write");
}

template <typename T>
int run_read(const ReadArgs &a, hipStream_t stream) {
    const int lanes = a.d <= 64 ? 4 : a.d <= 128 ? 8 : 16;
    const int64_t rows = (int64_t)a.length * a.kv_heads, blocks = (rows + kThreads / lanes - 1) / (kThreads / lanes);
    if (rows > INT32_MAX - kThreads || !kea::fits_dispatch(blocks, kThreads)) return kea::fail(KEA_EINVAL, "kea_paged_read: too large for one launch");
    const int64_t layers = (a.at.batch + 65534LL) / 65535;
    const dim3 grid((unsigned)blocks, (unsigned)((a.at.batch + layers - 1) / layers), (unsigned)(2 * layers));
    if (lanes == 4) read_kernel<T, 4><<<grid, kThreads, 0, stream>>>(a);
    else if (lanes == 8) read_kernel<T, 8><<<grid, kThreads, 0, stream>>>(a);
    else read_kernel<T, 16><<<grid, kThreads, 0, stream>>>(a);
    return launched("kea_paged_read");
}

}  // namespace

extern "C" {

int kea_paged_write(const kea_heads *k, const kea_heads *v, int dtype, int64_t kv_heads, int64_t d, const kea_pages *k_pages,
                    const kea_pages *v_pages, const kea_paging *paging, void *stream) {
    WriteArgs a{};
    const int rc = kea::check_paging("kea_paged_write", k_pages, v_pages, paging, kv_heads, d, &a.at);
    if (rc) return rc;
    if (!type_ok(dtype)) return kea::fail(KEA_EINVAL, "kea_paged_write: f32, f16 or bf16");
    const int64_t unit = dtype == KEA_F32 ? 4 : 8;
    if (!rows_ok(k, unit) || !rows_ok(v, unit)) return kea::fail(KEA_EALIGN, "kea_paged_write: tokens and their strides are multiples of 16 bytes, strides not negative");
    if (a.at.tokens == 0 || a.at.batch == 0 || a.at.width == 0 || a.at.pages == 0) return KEA_OK;
    if (!k->data_dev || !v->data_dev) return kea::fail(KEA_EINVAL, "kea_paged_write: a pointer is missing");
    a.k = *k, a.v = *v, a.kp = *k_pages, a.vp = *v_pages, a.kv_heads = (int)kv_heads, a.d = (int)d;
    const hipStream_t s = (hipStream_t)stream;
    return dtype == KEA_F32 ? run_write<float>(a, s) : dtype == KEA_F16 ? run_write<_Float16>(a, s) : run_write<__bf16>(a, s);
}

int kea_paged_read(const kea_pages *k_pages, const kea_pages *v_pages, const kea_paging *paging, const int32_t *starts, int64_t length,
                   int64_t kv_heads, int64_t d, void *k, void *v, int dtype, void *stream) {
    ReadArgs a{};
    kea_paging g = paging ? *paging : kea_paging{};
    g.tokens = 0, g.q_offsets_dev = nullptr;
    const int rc = kea::check_paging("kea_paged_read", k_pages, v_pages, paging ? &g : nullptr, kv_heads, d, &a.at);
    if (rc) return rc;
    if (!type_ok(dtype) || length < 0 || length > (1 << 30)) return kea::fail(KEA_EINVAL, "kea_paged_read: f32, f16 or bf16, and a length of 0 to 2^30");
    if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)starts % 4) return kea::fail(KEA_EALIGN, "kea_paged_read: outputs start at multiples of 16 bytes");
    if (length == 0 || a.at.batch == 0) return KEA_OK;
    if (!k || !v) return kea::fail(KEA_EINVAL, "kea_paged_read: a pointer is missing");
    a.kp = *k_pages, a.vp = *v_pages, a.starts = starts, a.k = k, a.v = v, a.kv_heads = (int)kv_heads, a.d = (int)d, a.length = (int)length;
    const hipStream_t s = (hipStream_t)stream;
    return dtype == KEA_F32 ? run_read<float>(a, s) : dtype == KEA_F16 ? run_read<_Float16>(a, s) : run_read<__bf16>(a, s);
}

}  // extern "C"
