// Writing tokens' keys and values to an int8 cache in pages, and reading them back (include/kea_decode.h).
//
//   s = max(max|x| / 127, 1e-30), held to where 127 s is finite, c = rint(x / s) for each row x of d elements;   x' = c s
//
// Either moves bytes and little else: a wave takes one token or position, whose sequence and page are then uniform, and runs
// through its 2 kv_heads rows, L = 8, 16 or 32 lanes of eight elements to a row.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_internal.h"
#include "kea_pages.h"
#include "kea_rowq.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint16_t v8u __attribute__((ext_vector_type(8)));

constexpr float kMostScale = 0x1.0204060000000p+121f;  // the largest s of which 127 s is a finite number
constexpr int kWaves = 4;  // tokens or positions of a workgroup

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
    v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));  // the other four of eight
    if constexpr (L >= 16) v = max(v, dpp(v, std::integral_constant<int, 0x140>{}));  // the other eight of 16
    if constexpr (L >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    return v;
}

struct WriteArgs {
    kea_heads k, v;
    kea_pages kp, vp;
    kea::Paging at;
    int kv_heads, d;
};

// U passes of 64 / L rows each are loaded at once.
template <typename T, int L, int U>
__global__ void __launch_bounds__(64 * kWaves) write_kernel(WriteArgs a) {
    const int lane = threadIdx.x & 63, t = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    if (t >= a.at.tokens) return;
    const int b = a.at.sequence(t);
    if (b < 0) return;
    const int2 rows = a.at.rows(b);
    const int p = a.at.length(b) - rows.y + t;  // len - n + i
    if (p < 0) return;
    const int page = __builtin_amdgcn_readfirstlane(a.at.page(b, p));
    if (page < 0) return;
    const int row = p & ((1 << a.at.shift) - 1), at = lane % L * 8;
    for (int r0 = 0; r0 < 2 * a.kv_heads; r0 += U * (64 / L)) {
        float x[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * (64 / L) + lane / L, h = r >> 1;
            const kea_heads &from = r & 1 ? a.v : a.k;
            if (h < a.kv_heads && at < a.d) load8((const T *)from.data_dev + (long long)t * from.t_stride + (long long)h * from.head_stride + at, x[u]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) x[u][e] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * (64 / L) + lane / L, h = r >> 1;
            const kea_pages &to = r & 1 ? a.vp : a.kp;
            uint32_t most = 0;  // (as whole numbers the sizes keep their order, with infinities and NaN on top)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, __builtin_bit_cast(uint32_t, x[u][e]) & 0x7FFFFFFFu);
            most = lanes_max<L>(most);
            const bool number = most < 0x7F800000u;
            const float s = number ? fminf(fmaxf(__builtin_bit_cast(float, most) / 127.0f, 1e-30f), kMostScale) : __builtin_nanf(""), inv = 1.0f / s;
            uint32_t code[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float z = x[u][e];
                code[e] = number ? kea::quantize_code(z, s, inv) : 0u;
            }
            if (h < a.kv_heads && at < a.d) {
                v2u w;
#pragma unroll
                for (int i = 0; i < 2; ++i) w[i] = code[4 * i] | code[4 * i + 1] << 8 | code[4 * i + 2] << 16 | code[4 * i + 3] << 24;
                *(v2u *)(to.data_dev + page * to.page_stride + h * to.head_stride + row * to.row_stride + at) = w;
                if (at == 0) to.scale_dev[page * to.scale_page_stride + h * to.scale_head_stride + row * to.scale_row_stride] = s;
            }
        }
    }
}

struct ReadArgs {
    kea_pages kp, vp;
    kea::Paging at;
    const int32_t *starts;
    void *k, *v;
    int kv_heads, d, length;
};

template <typename T, int L, int U>
__global__ void __launch_bounds__(64 * kWaves) read_kernel(ReadArgs a) {
    const int lane = threadIdx.x & 63, i = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6)), b = blockIdx.y;
    if (i >= a.length) return;
    const long long p = (a.starts ? (long long)a.starts[b] : 0) + i;
    const int page = __builtin_amdgcn_readfirstlane(p >= 0 && p < a.at.length(b) ? a.at.page(b, (int)p) : -1);
    const int row = (int)p & ((1 << a.at.shift) - 1), at = lane % L * 8;
    const long long out = ((long long)b * a.length + i) * a.kv_heads * a.d;
    for (int r0 = 0; r0 < 2 * a.kv_heads; r0 += U * (64 / L)) {
        v2u c[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * (64 / L) + lane / L, h = r >> 1;
            const kea_pages &from = r & 1 ? a.vp : a.kp;
            c[u] = v2u{0, 0};
            s[u] = 0.0f;
            if (page >= 0 && h < a.kv_heads && at < a.d) {
                c[u] = *(const v2u *)(from.data_dev + page * from.page_stride + h * from.head_stride + row * from.row_stride + at);
                s[u] = from.scale_dev[page * from.scale_page_stride + h * from.scale_head_stride + row * from.scale_row_stride];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * (64 / L) + lane / L, h = r >> 1;
            if (h >= a.kv_heads || at >= a.d) continue;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)(c[u][e / 4] >> (8 * (e % 4))) * s[u];
            store8((T *)(r & 1 ? a.v : a.k) + out + (long long)h * a.d + at, x);
        }
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
    const dim3 grid((unsigned)((a.at.tokens + kWaves - 1) / kWaves));
    if (!kea::fits_dispatch(grid.x, 64 * kWaves)) return kea::fail(KEA_EINVAL, "kea_paged_write: too large for one launch");
    if (a.d <= 64) write_kernel<T, 8, 2><<<grid, 64 * kWaves, 0, stream>>>(a);
    else if (a.d <= 128) write_kernel<T, 16, 2><<<grid, 64 * kWaves, 0, stream>>>(a);
    else write_kernel<T, 32, 2><<<grid, 64 * kWaves, 0, stream>>>(a);
    return launched("kea_paged_write");
}

template <typename T>
int run_read(const ReadArgs &a, hipStream_t stream) {
    const dim3 grid((unsigned)((a.length + kWaves - 1) / kWaves), (unsigned)a.at.batch);
    if (!kea::fits_dispatch(grid.x, 64 * kWaves) || a.at.batch > 65535) return kea::fail(KEA_EINVAL, "kea_paged_read: too large for one launch");
    if (a.d <= 64) read_kernel<T, 8, 2><<<grid, 64 * kWaves, 0, stream>>>(a);
    else if (a.d <= 128) read_kernel<T, 16, 2><<<grid, 64 * kWaves, 0, stream>>>(a);
    else read_kernel<T, 32, 2><<<grid, 64 * kWaves, 0, stream>>>(a);
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
