// Attention within a sliding window and to the first tokens (include/kea_block.h): one wave per query and head, key by key
// with a running maximum and sum, each lane holding up to four of the head's elements.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_internal.h"
#include "kea_wave.h"
#include "../../include/kea_block.h"

namespace {

struct Args {
    kea_heads q, k, v, out;
    const int32_t *lengths, *starts;
    long long rows;
    int tq, tk, heads, group, d, left, right, sinks, dtype;
    float scale;
};

__device__ __forceinline__ float load(const void *p, int dtype, long long i) {
    if (dtype == KEA_F32) return ((const float *)p)[i];
    if (dtype == KEA_F16) return (float)((const _Float16 *)p)[i];
    return (float)((const __bf16 *)p)[i];
}

__global__ void __launch_bounds__(256) window_kernel(Args a) {
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    const int lane = threadIdx.x & 63;
    const int h = (int)(row % a.heads), t = (int)(row / a.heads % a.tq);
    const long long b = row / a.heads / a.tq;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.tk) : a.tk;
    const int start = a.starts ? min(max(a.starts[b], -(1 << 30)), 1 << 30) : len - a.tq;
    const int p = start + t;
    const long long qo = b * a.q.batch_stride + t * a.q.t_stride + h * a.q.head_stride;
    const long long ko = b * a.k.batch_stride + h / a.group * a.k.head_stride;
    const long long vo = b * a.v.batch_stride + h / a.group * a.v.head_stride;
    float q[4], o[4] = {0, 0, 0, 0}, top = -INFINITY, sum = 0.0f;
    for (int e = 0; e < 4; ++e) q[e] = lane + 64 * e < a.d ? load(a.q.data_dev, a.dtype, qo + lane + 64 * e) * a.scale : 0.0f;
    if (p >= 0 && p < len) {
        const int low = max(0, p - a.left), high = min(len - 1, (int)min((long long)p + a.right, 1LL << 30));
        const int first = min(min(a.sinks, low), high + 1);
        for (int i = 0; i < first + (high - low + 1); ++i) {
            const int j = i < first ? i : low + (i - first);
            float s = 0.0f;
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < a.d) s += q[e] * load(a.k.data_dev, a.dtype, ko + j * a.k.t_stride + lane + 64 * e);
            s = kea::wave_sum(s);
            const float next = fmaxf(top, s), old = top == -INFINITY ? 0.0f : expf(top - next);
            const float w = s == -INFINITY ? 0.0f : expf(s - next);
            top = next;
            sum = sum * old + w;
            for (int e = 0; e < 4; ++e)
                o[e] = o[e] * old + (lane + 64 * e < a.d ? w * load(a.v.data_dev, a.dtype, vo + j * a.v.t_stride + lane + 64 * e) : 0.0f);
        }
    }
    const long long oo = b * a.out.batch_stride + t * a.out.t_stride + h * a.out.head_stride;
    for (int e = 0; e < 4; ++e) {
        if (lane + 64 * e >= a.d) break;
        const float v = sum != 0.0f ? o[e] / sum : 0.0f;
        const long long at = oo + lane + 64 * e;
        if (a.dtype == KEA_F32) ((float *)a.out.data_dev)[at] = v;
        else if (a.dtype == KEA_F16) ((_Float16 *)a.out.data_dev)[at] = (_Float16)v;
        else ((__bf16 *)a.out.data_dev)[at] = (__bf16)v;
    }
}

bool heads_ok(const kea_heads *t, int64_t unit) {
    return t && (uintptr_t)t->data_dev % 16 == 0 && t->batch_stride % unit == 0 && t->t_stride % unit == 0 && t->head_stride % unit == 0;
}

int check_sizes(const char *what, int dtype, int64_t batch, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d,
                int64_t left, int64_t right, int64_t sinks) {
    if (dtype != KEA_F32 && dtype != KEA_F16 && dtype != KEA_BF16) return kea::fail(KEA_EINVAL, std::string(what) + ": f32, f16 or bf16");
    if (batch < 0 || tq < 0 || tk < 0 || tq > (1 << 30) || tk > (1 << 30) || heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 65535)
        return kea::fail(KEA_EINVAL, std::string(what) + ": batch >= 0, 0 <= tq, tk <= 2^30 and heads a multiple of kv_heads are needed");
    if (d < 8 || d > 256 || d % 8) return kea::fail(KEA_EINVAL, std::string(what) + ": d is a multiple of 8 from 8 to 256");
    if (left < 0 || right < 0 || sinks < 0) return kea::fail(KEA_EINVAL, std::string(what) + ": left, right and sinks are >= 0");
    return KEA_OK;
}

}  // namespace

extern "C" {

int64_t kea_window_attention_workspace(int dtype, int64_t batch, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d,
                                       int64_t left, int64_t right, int64_t sinks) {
    return check_sizes("kea_window_attention_workspace", dtype, batch, tq, tk, heads, kv_heads, d, left, right, sinks);
}

int kea_window_attention(const kea_heads *q, const kea_heads *k, const kea_heads *v, const kea_heads *out, int dtype, int64_t batch,
                         int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d, int64_t left, int64_t right,
                         int64_t sinks, float scale, const int32_t *kv_lengths, const int32_t *q_starts, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    const int rc = check_sizes("kea_window_attention", dtype, batch, tq, tk, heads, kv_heads, d, left, right, sinks);
    if (rc) return rc;
    const int64_t unit = dtype == KEA_F32 ? 4 : 8;
    if (!heads_ok(q, unit) || !heads_ok(k, unit) || !heads_ok(v, unit) || !heads_ok(out, unit) || (uintptr_t)kv_lengths % 4 || (uintptr_t)q_starts % 4)
        return kea::fail(KEA_EALIGN, "kea_window_attention: pointers and strides are multiples of 16 bytes");
    if (batch == 0 || tq == 0) return KEA_OK;
    if (!q->data_dev || !out->data_dev || (tk > 0 && (!k->data_dev || !v->data_dev))) return kea::fail(KEA_EINVAL, "kea_window_attention: a pointer is missing");
    const int64_t most = 1 << 30, rows = batch * tq * heads;
    Args a{*q, *k, *v, *out, kv_lengths, q_starts, rows, (int)tq, (int)tk, (int)heads, (int)(heads / kv_heads), (int)d,
           (int)(left < most ? left : most), (int)(right < most ? right : most), (int)(sinks < most ? sinks : most), dtype, scale};
    if (batch > most || !kea::fits_dispatch((rows + 3) / 4, 256)) return kea::fail(KEA_EINVAL, "kea_window_attention: too large for one launch");
    window_kernel<<<dim3((unsigned)((rows + 3) / 4)), 256, 0, (hipStream_t)stream>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_window_attention: ") + hipGetErrorString(e));
}

}  // extern "C"
