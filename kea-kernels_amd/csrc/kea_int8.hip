// int8 x int8 matrix product with a scale for each token and channel (include/kea_block.h).
//
//   acc[m][n] = sum_k q[m][k] w[n][k]   on v_mfma_i32_16x16x64_i8, then the epilogue of kea_epilogue.h
//
// The weight rows are the instruction's first operand, so lane 16 g + i ends up with columns 4 g .. 4 g + 3 of output row
// i of a 16 x 16 block. Bytes of q from k on are masked to zero, so what w holds there does not matter.
//
// Two kernels:
//   tile_kernel   many output tiles: a workgroup owns BM x BN outputs; stages of 128 k of both operands stream into LDS by
//                 direct copies, NS stages deep, and every byte is read by several waves. 16000 x 4096 x 4096 in 256 x 256
//                 tiles takes 233 us, 2.3 POP/s of the 4.1 that the int8 matrix instruction reaches on such data (a library
//                 product of that size 255): the matrix cores wait at the barrier of each stage, when all eight waves read
//                 their next operands at once; reading one tile's operands for all tiles, out of L2, takes as long.
//   split_kernel  few output tiles (few tokens): a workgroup owns 16 RM x 16 RN outputs, its NW waves share out k, each
//                 loading its operands straight into registers, and the exact int32 sums meet in LDS. 1 x 2560 x 640 takes
//                 3.8 us, of which an empty launch is 1.6; 16 x 1024 x 4096 6.6, the time in which one workgroup takes in the
//                 128 KB that it needs, be they 64 of them or 256 (64 x 1024 x 4096: 5.9).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "kea_epilogue.h"
#include "kea_internal.h"
#include "../../include/kea_block.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
// Rows of outputs and of the residual start at any element: vectors of them, aligned to an element. (Global memory takes
// such accesses whole.)
typedef int32_t i32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8), aligned(2)));

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

// ---- epilogue ----------------------------------------------------------------------------------------------------------------

// Element i of a vector of FP32 or FP16 values, without a branch on its type: the aligned word that holds it, and its value
// from that word. 0 without a vector.
__device__ __forceinline__ uint32_t scalar_word(const void *p, int dtype, int i) {
    const uintptr_t at = (uintptr_t)p + (dtype == KEA_F16 ? 2 : 4) * (uintptr_t)i;
    return p ? *(const __attribute__((address_space(1))) uint32_t *)(at & ~(uintptr_t)3) : 0u;
}
__device__ __forceinline__ float scalar_value(uint32_t word, const void *p, int dtype, int i) {
    const uint32_t half = ((uintptr_t)p + 2 * (uintptr_t)i) & 2 ? word >> 16 : word & 0xFFFFu;
    return dtype == KEA_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)half) : __builtin_bit_cast(float, word);
}

// Scales and bias of four consecutive columns.
struct Columns {
    float a[4], b[4];
};
__device__ __forceinline__ Columns columns(const Args &p, int n0) {
    Columns c;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int n = min(n0 + r, p.n - 1);
        c.a[r] = p.ws ? kea::load_scalar(p.ws, p.ws_dtype, n) : 0.0f;
        c.b[r] = p.bias ? kea::load_scalar(p.bias, p.bias_dtype, n) : kea::kNoBias;
    }
    return c;
}

// Outputs [row][n0 .. n0 + 3] from their sums; s the row's scale.
__device__ __forceinline__ void store4(const Args &p, int row, int n0, v4i acc, float s, const Columns &c) {
    const long long at = (long long)row * p.ldy + n0;
    const bool full = n0 + 3 < p.n;
    if (p.y_dtype == KEA_I32) {
        int32_t *y = (int32_t *)p.y + at;
        if (full) *(i32x4 *)y = acc;
        else
            for (int r = 0; r < 4; ++r)
                if (n0 + r < p.n) y[r] = acc[r];
        return;
    }
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = kea::finish((float)acc[r] * s, c.a[r], c.b[r], p.flags);
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

// Outputs [row][n0 .. n0 + 7] from their sums, in two halves; a and b the columns' scales and biases.
__device__ __forceinline__ void store8(const Args &p, int row, int n0, v4i lo, v4i hi, float s, const float *a, const float *b) {
    if (n0 + 7 >= p.n) {
        Columns c;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (n0 + 4 * half >= p.n) break;
#pragma unroll
            for (int r = 0; r < 4; ++r) c.a[r] = a[4 * half + r], c.b[r] = b[4 * half + r];
            store4(p, row, n0 + 4 * half, half ? hi : lo, s, c);
        }
        return;
    }
    char *const y = (char *)p.y;
    const long long at = (long long)row * p.ldy + n0;
    if (p.y_dtype == KEA_I32) {
        *(i32x4 *)(y + 4 * at) = lo;
        *(i32x4 *)(y + 4 * at + 16) = hi;
        return;
    }
    float v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = __builtin_fmaf((float)(r < 4 ? lo[r & 3] : hi[r & 3]) * s, a[r], b[r]);
    if (p.flags & KEA_FLAG_SILU)
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = kea::silu_epilogue(v[r]);
    if (p.res) {
        const float *res = p.res + (long long)row * p.ldr + n0;
        const f32x4 x[2] = {*(const f32x4 *)res, *(const f32x4 *)(res + 4)};
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = x[r / 4][r % 4] + v[r] * p.factor;
    }
    if (p.y_dtype == KEA_F32) {
        *(f32x4 *)(y + 4 * at) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4 *)(y + 4 * at + 16) = f32x4{v[4], v[5], v[6], v[7]};
        return;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) asm("" : "+v"(v[r]));  // rounded to FP32 before they are rounded to 16 bits
    if (p.y_dtype == KEA_F16) {
        *(f16x8 *)(y + 2 * at) = f16x8{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3], (_Float16)v[4], (_Float16)v[5], (_Float16)v[6], (_Float16)v[7]};
    } else {
        *(bf16x8 *)(y + 2 * at) = bf16x8{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3], (__bf16)v[4], (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]};
    }
}

// Sixteen bytes of a row of k elements that start at k0, those from k on set to zero.
__device__ __forceinline__ v4i mask16(v4i v, int k0, int k) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int left = k - (k0 + 4 * d);
        if (left < 4) v[d] = left <= 0 ? 0 : v[d] & ((1 << (8 * left)) - 1);
    }
    return v;
}

// ---- many tiles ----------------------------------------------------------------------------------------------------------------

typedef __attribute__((address_space(1))) const void *gptr_t;
typedef __attribute__((address_space(3))) void *lptr_t;

template <int N>
__device__ __forceinline__ void wait_copies() {  // at most N of this wave's copies outstanding (vmcnt), none of its LDS reads
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// BK bytes of k a stage. LDS holds a stage's rows of BK bytes in 16-byte units, unit c of row r at place c ^ f(r): the rows
// that one operand read takes lie in different banks.
//
// Which weight rows make up a 16-row operand is free: operands 2 j and 2 j + 1 of a wave take 8 (i / 4) + i % 4 and the same
// + 4 of its columns 32 j .. 32 j + 31, so that a lane's sums of the two are eight consecutive columns, and the four lanes of
// a row store 32.
template <int BM, int BN, int WM, int WN, int BK, int NS>
__global__ void __launch_bounds__(WM *WN * 64) tile_kernel(Args p, int tiles_m, int tiles_n) {
    constexpr int NT = WM * WN * 64, RM = BM / WM / 16, RN = BN / WN / 16, UNITS = BK / 16;
    constexpr int CA = BM * UNITS / NT, CB = BN * UNITS / NT, COPIES = CA + CB;  // copies of a stage by each thread
    constexpr int STAGE = (BM + BN) * BK;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *const row_scale = (float *)(lds + NS * STAGE), *const col_scale = row_scale + BM, *const col_bias = col_scale + BN;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15, wm = wave / WN, wn = wave % WN;

    // Workgroups go to the eight XCDs in turn; each XCD takes a run of tiles of its own, in groups of 8 tiles of rows that
    // share their columns, so that what runs at once shares operands in that XCD's L2.
    const int total = tiles_m * tiles_n, per = total / 8, rest = total % 8, x = blockIdx.x % 8;
    const int id = x * per + min(x, rest) + blockIdx.x / 8;
    const int band = id / (8 * tiles_n), in = id % (8 * tiles_n), rows = min(8, tiles_m - 8 * band);
    const int m0 = (8 * band + in % rows) * BM, n0 = in / rows * BN;

    // swizzle of a row of q and of w: over the eight rows that eight lanes of a read take
    auto fq = [](int r) { return UNITS == 8 ? r & 7 : (r >> 1) & 3; };
    auto fw = [](int r) { return UNITS == 8 ? (r >> 3 & 1) * 4 + (r & 3) : (r >> 3 & 1) * 2 + (r >> 1 & 1); };
    // the copies of this thread: unit tid + u NT of a stage's rows, the same unit of a row for every u
    static_assert(NT / UNITS % 16 == 0 && RN % 2 == 0, "the swizzles repeat from copy to copy");
    const int unit_q = ((tid % UNITS) ^ fq(tid / UNITS)) * 16, unit_w = ((tid % UNITS) ^ fw(tid / UNITS)) * 16;
    uint32_t at[COPIES];
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
        const int r = tid / UNITS + (u < CA ? u : u - CA) * (NT / UNITS);
        at[u] = u < CA ? (uint32_t)min(r, p.m - 1 - m0) * (uint32_t)p.ldq + unit_q : (uint32_t)min(r, p.n - 1 - n0) * (uint32_t)p.ldw + unit_w;
    }
    const int8_t *const q0 = p.q + (long long)m0 * p.ldq, *const w0 = p.w + (long long)n0 * p.ldw;
    const int last = (p.k - 1) & ~15, stages = (p.k + BK - 1) / BK;  // the last unit of a row
    static_assert(BK == 128, "a stage is two steps of 64");
    auto copy = [&](int s, int buf) {
        // units past the row's end are read from its last one
        const int back_q = min(0, last - (s * BK + unit_q)), back_w = min(0, last - (s * BK + unit_w));
#pragma unroll
        for (int u = 0; u < COPIES; ++u)
            __builtin_amdgcn_global_load_lds((gptr_t)((u < CA ? q0 : w0) + s * BK + (size_t)(at[u] + (uint32_t)(u < CA ? back_q : back_w))),
                                             (lptr_t)(lds + buf * STAGE + (u < CA ? 0 : BM * BK) + ((u < CA ? u : u - CA) * NT + wave * 64) * 16), 16, 0, 0);
    };
    // The last stage's bytes of q from k on become zeros (once they have landed; all waves pass here together).
    auto clear_tail = [&](int s, int buf) {
        if ((s + 1) * BK <= p.k) return;
#pragma unroll
        for (int u = 0; u < CA; ++u) {
            v4i *const v = (v4i *)(lds + buf * STAGE + (u * NT + tid) * 16);
            *v = mask16(*v, s * BK + unit_q, p.k);
        }
        __syncthreads();
    };

    v4i acc[RM][RN];
#pragma unroll
    for (int a = 0; a < RM; ++a)
#pragma unroll
        for (int b = 0; b < RN; ++b) acc[a][b] = v4i{0, 0, 0, 0};

    const int wrow = 8 * (i >> 2) + (i & 3);
    v4i qf[2][RM], wf[2][RN];
    auto fetch = [&](int buf, int h, int set) {
        const char *qa = lds + buf * STAGE + (wm * RM * 16 + i) * BK, *wa = lds + buf * STAGE + (BM + wn * RN * 16 + wrow) * BK;
        const int pq = ((4 * h + g) ^ fq(i)) * 16, pw = ((4 * h + g) ^ fw(wrow)) * 16;
#pragma unroll
        for (int b = 0; b < RN; ++b) wf[set][b] = *(const v4i *)(wa + (b / 2 * 32 + b % 2 * 4) * BK + pw);
#pragma unroll
        for (int a = 0; a < RM; ++a) qf[set][a] = *(const v4i *)(qa + a * 16 * BK + pq);
    };
    auto product = [&](int set) {
#pragma unroll
        for (int a = 0; a < RM; ++a)
#pragma unroll
            for (int b = 0; b < RN; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[set][b], qf[set][a], acc[a][b], 0, 0, 0);
    };
    // scales and bias of the tile, on their way while the first copies are issued
    constexpr int LR = (BM + NT - 1) / NT, LC = (BN + NT - 1) / NT;
    uint32_t rs[LR], cs[LC], cb[LC];
#pragma unroll
    for (int u = 0; u < LR; ++u) rs[u] = scalar_word(p.qs, p.qs_dtype, min(m0 + tid + u * NT, p.m - 1));
#pragma unroll
    for (int u = 0; u < LC; ++u) {
        cs[u] = scalar_word(p.ws, p.ws_dtype, min(n0 + tid + u * NT, p.n - 1));
        cb[u] = scalar_word(p.bias, p.bias_dtype, min(n0 + tid + u * NT, p.n - 1));
    }
    // With two buffers a stage's copies start as soon as the waves have read what its buffer held, in the middle of a stage;
    // with more there is time, and they start with the next stage, off the operands' way (NS = 2: 16000 x 4096 x 4096 250 -> 231
    // us, NS = 4: 1000 x 1024 x 4096 11.2 -> 10.7).
    constexpr bool MIDDLE = NS == 2;
    constexpr int AHEAD = MIDDLE ? NS : NS - 1;
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) copy(min(s, stages - 1), s);
#pragma unroll
    for (int u = 0; u < LR; ++u)
        if (tid + u * NT < BM) row_scale[tid + u * NT] = scalar_value(rs[u], p.qs, p.qs_dtype, min(m0 + tid + u * NT, p.m - 1));
#pragma unroll
    for (int u = 0; u < LC; ++u)
        if (tid + u * NT < BN) {
            col_scale[tid + u * NT] = scalar_value(cs[u], p.ws, p.ws_dtype, min(n0 + tid + u * NT, p.n - 1));
            col_bias[tid + u * NT] = p.bias ? scalar_value(cb[u], p.bias, p.bias_dtype, min(n0 + tid + u * NT, p.n - 1)) : kea::kNoBias;
        }
    wait_copies<(AHEAD - 1) * COPIES>();
    barrier();
    if (stages == 1) clear_tail(0, 0);
    fetch(0, 0, 0);
    // Stage s, whose first half's operands are in set 0: each half's operands are read while the matrix cores work on the
    // other's. Between its halves the next stage has landed. (Past the end the last stage is copied again: every wave counts
    // the same copies.)
    int buf = 0;
    for (int s = 0; s + 1 < stages; ++s) {
        if (!MIDDLE) copy(min(s + AHEAD, stages - 1), buf ? buf - 1 : NS - 1);
        fetch(buf, 1, 1);
        product(0);
        wait_copies<(NS - 2) * COPIES>();
        barrier();
        if (MIDDLE) copy(min(s + AHEAD, stages - 1), buf);
        buf = buf + 1 == NS ? 0 : buf + 1;
        if (s + 2 == stages) clear_tail(s + 1, buf);
        fetch(buf, 0, 0);
        product(1);
    }
    fetch(buf, 1, 1);
    product(0);
    product(1);
    wait_copies<0>();

#pragma unroll
    for (int b = 0; b < RN; b += 2) {
        const int c0 = (wn * RN + b) * 16 + 8 * g;
        if (n0 + c0 >= p.n) continue;
        float ca[8], cb[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) ca[r] = col_scale[c0 + r], cb[r] = col_bias[c0 + r];
#pragma unroll
        for (int a = 0; a < RM; ++a) {
            const int r = (wm * RM + a) * 16 + i;
            if (m0 + r < p.m) store8(p, m0 + r, n0 + c0, acc[a][b], acc[a][b + 1], row_scale[r], ca, cb);
        }
    }
}

// ---- few tiles -----------------------------------------------------------------------------------------------------------------

template <int RM, int RN, int NW, int U>  // U: k-steps of 64 loaded at once
__global__ void __launch_bounds__(NW * 64) split_kernel(Args p, int tiles_n) {
    static_assert(RM * RN <= NW, "a wave finishes one block at most");
    __shared__ v4i part[NW][RM * RN][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
    const int m0 = blockIdx.x / tiles_n * (16 * RM), n0 = blockIdx.x % tiles_n * (16 * RN);
    const int steps = (p.k + 63) / 64, from = (int)((long long)steps * wave / NW), to = (int)((long long)steps * (wave + 1) / NW);
    const int last = (p.k - 1) & ~15;
    const int8_t *qr[RM], *wr[RN];
#pragma unroll
    for (int a = 0; a < RM; ++a) qr[a] = p.q + (long long)min(m0 + 16 * a + i, p.m - 1) * p.ldq;
#pragma unroll
    for (int b = 0; b < RN; ++b) wr[b] = p.w + (long long)min(n0 + 16 * b + i, p.n - 1) * p.ldw;
    v4i acc[RM][RN];
#pragma unroll
    for (int a = 0; a < RM; ++a)
#pragma unroll
        for (int b = 0; b < RN; ++b) acc[a][b] = v4i{0, 0, 0, 0};
    v4i qf[U][RM], wf[U][RN];
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(64 * (s0 + u) + 16 * g, last);
#pragma unroll
            for (int b = 0; b < RN; ++b) wf[u][b] = *(const v4i *)(wr[b] + at);
#pragma unroll
            for (int a = 0; a < RM; ++a) qf[u][a] = *(const v4i *)(qr[a] + at);
        }
    };
    auto product = [&](int s0) {
        const int end = min(p.k, 64 * to);  // (steps past this wave's share are masked like those past k)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = 64 * (s0 + u) + 16 * g;
            if (64 * (s0 + u) + 64 > end)
#pragma unroll
                for (int a = 0; a < RM; ++a) qf[u][a] = mask16(qf[u][a], at, end);
#pragma unroll
            for (int a = 0; a < RM; ++a)
#pragma unroll
                for (int b = 0; b < RN; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][b], qf[u][a], acc[a][b], 0, 0, 0);
        }
    };
    // the first operands, then the scales and bias of the block that this wave finishes: on their way together
    load(from);
    const int row = m0 + wave / RN % RM * 16 + i, col = n0 + wave % RN * 16 + 4 * g;
    const int srow = min(row, p.m - 1);
    const uint32_t rs = scalar_word(p.qs, p.qs_dtype, srow);
    uint32_t cs[4], cb[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        cs[r] = scalar_word(p.ws, p.ws_dtype, min(col + r, p.n - 1));
        cb[r] = scalar_word(p.bias, p.bias_dtype, min(col + r, p.n - 1));
    }
    product(from);
    for (int s0 = from + U; s0 < to; s0 += U) {
        load(s0);
        product(s0);
    }
#pragma unroll
    for (int a = 0; a < RM; ++a)
#pragma unroll
        for (int b = 0; b < RN; ++b) part[wave][a * RN + b][lane] = acc[a][b];
    __syncthreads();
    if (wave >= RM * RN || row >= p.m || col >= p.n) return;
    v4i sum = part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) sum += part[w][wave][lane];
    Columns c;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        c.a[r] = scalar_value(cs[r], p.ws, p.ws_dtype, min(col + r, p.n - 1));
        c.b[r] = p.bias ? scalar_value(cb[r], p.bias, p.bias_dtype, min(col + r, p.n - 1)) : kea::kNoBias;
    }
    store4(p, row, col, sum, scalar_value(rs, p.qs, p.qs_dtype, srow), c);
}

// ---- host ----------------------------------------------------------------------------------------------------------------------

bool scale_type(int t) { return t == KEA_F32 || t == KEA_F16; }
bool aligned(const void *p, int dtype) { return (uintptr_t)p % (dtype == KEA_F32 || dtype == KEA_I32 ? 4 : 2) == 0; }

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string(what) + ": " + hipGetErrorString(e));
}

template <int BM, int BN, int WM, int WN, int BK, int NS>
int run_tiles(const Args &a, hipStream_t stream) {
    constexpr int lds = NS * (BM + BN) * BK + (BM + 2 * BN) * 4;
    static_assert(lds <= 160 * 1024 && BM * BK / 16 % (WM * WN * 64) == 0 && BN * BK / 16 % (WM * WN * 64) == 0, "stage buffers and copies");
    const int tm = (a.m + BM - 1) / BM, tn = (a.n + BN - 1) / BN;
    const long long tiles = (long long)tm * tn;
    if (tiles > INT32_MAX / 2 || !kea::fits_dispatch(tiles, WM * WN * 64)) return kea::fail(KEA_EINVAL, "kea_int8_gemm: too large for one launch");
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)tile_kernel<BM, BN, WM, WN, BK, NS>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return kea::fail((int)e, std::string("kea_int8_gemm: ") + hipGetErrorString(e));
    }
    tile_kernel<BM, BN, WM, WN, BK, NS><<<dim3((unsigned)tiles), WM * WN * 64, lds, stream>>>(a, tm, tn);
    return launched("kea_int8_gemm");
}

template <int RM, int RN, int NW, int U>
int run_split(const Args &a, hipStream_t stream) {
    const int tn = (a.n + 16 * RN - 1) / (16 * RN);
    const long long tiles = (long long)((a.m + 16 * RM - 1) / (16 * RM)) * tn;
    if (tiles > INT32_MAX / 2 || !kea::fits_dispatch(tiles, NW * 64)) return kea::fail(KEA_EINVAL, "kea_int8_gemm: too large for one launch");
    split_kernel<RM, RN, NW, U><<<dim3((unsigned)tiles), NW * 64, 0, stream>>>(a, tn);
    return launched("kea_int8_gemm");
}

// The variant of the shortest estimated time. Each tile form's launch takes `base` us and, for every `full` workgroups that
// run at once, fa us a stage of 128 k and fe besides (ha and he where at most 256 are left, one to a CU); the forms that split
// k take what the bytes of one workgroup take (they are too few to fill the CU's loads) or, with many workgroups, what all take.
// The figures are fits to what the forms take on 60 shapes of 1 to 16000 rows, hot, as graphs of launches; some of them (us, the
// tile forms in the order below, then 32 x 32, 32 x 16 and 16 x 16 split over 4 waves):
//   8000 x 4096 x 4096   116.7  138.4  159.2  173.6  232.1
//   2000 x 4096 x 1024    19.4   14.4   15.9   16.6   21.9
//   1000 x 4096 x 1024    17.2    8.6    8.4    9.1   12.3  31.7
//   1500 x 1024 x 1024    16.4    7.4    7.3    5.7    6.3  13.5
//   1000 x 1024 x 1024    16.1    7.2    7.1    5.5    4.9   9.9
//    125 x 1024 x 1024    15.2    6.9    6.8    5.1    4.5   4.3    3.6    4.0
//     64 x 4096 x 1024    13.4    6.8    6.8    5.1    4.5   4.4    5.3    5.9
//     16 x 2560 x  640     9.1    4.7    4.9    3.9    3.7   3.6    3.4    3.2
//     64 x 1024 x 4096    40.1   17.0   16.1   11.5    9.8   9.4    7.7    5.9
struct Form {
    int bm, bn, full;
    float base, fa, fe, ha, he;
};
constexpr Form kForms[] = {{256, 256, 256, 2.0f, 1.45f, 8.0f, 1.45f, 8.0f},
                           {128, 128, 512, 2.3f, 0.93f, 3.2f, 0.62f, 1.3f},
                           {128, 128, 256, 2.0f, 0.48f, 2.9f, 0.48f, 2.9f},
                           {128, 64, 512, 2.0f, 0.55f, 2.7f, 0.36f, 1.3f},
                           {64, 64, 512, 2.0f, 0.37f, 1.9f, 0.23f, 1.1f}};
constexpr int kSplit32 = 5, kSplit32x16 = 6, kSplit16 = 7;

int choose(int m, int n, int k) {
    auto tiles = [&](int bm, int bn) { return (double)((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
    const float stages = (float)((k + 127) / 128);
    int best = kSplit16;
    double least = 1e30;
    auto take = [&](int v, double t) {
        if (t < least) least = t, best = v;
    };
    auto split = [&](int v, int bm, int bn, double one, double all) {
        const double a = 2.4 + one * stages, b = 2.5 + all * stages * tiles(bm, bn);
        take(v, a > b ? a : b);
    };
    split(kSplit16, 16, 16, 0.11, 0.00045);
    split(kSplit32x16, 32, 16, 0.165, 0.00064);
    split(kSplit32, 32, 32, 0.22, 0.001);
    for (int v = 0; v < (int)(sizeof(kForms) / sizeof(kForms[0])); ++v) {
        const Form &f = kForms[v];
        const double t = tiles(f.bm, f.bn), rounds = (double)(long long)(t / f.full), left = t - rounds * f.full;
        take(v, f.base + rounds * (f.fa * stages + f.fe) + (left > 256 ? f.fa * stages + f.fe : left > 0 ? f.ha * stages + f.he : 0));
    }
    return best;
}

int run(int variant, const Args &a, hipStream_t stream) {
    switch (variant) {
        case 0: return run_tiles<256, 256, 2, 4, 128, 2>(a, stream);
        case 1: return run_tiles<128, 128, 2, 4, 128, 2>(a, stream);
        case 2: return run_tiles<128, 128, 2, 4, 128, 4>(a, stream);
        case 3: return run_tiles<128, 64, 4, 2, 128, 3>(a, stream);
        case 4: return run_tiles<64, 64, 4, 2, 128, 4>(a, stream);
        case kSplit32: return run_split<2, 2, 4, 2>(a, stream);
        case kSplit32x16: return run_split<2, 1, 4, 4>(a, stream);
        case kSplit16: return run_split<1, 1, 4, 4>(a, stream);
        default: return kea::fail(KEA_EINVAL, "kea_int8_gemm: no such variant");
    }
}

}  // namespace

extern "C" {

int kea_int8_gemm(const int8_t *q, int64_t ldq, const void *qs, int qs_dtype, const int8_t *w, int64_t ldw, const void *wscale,
                  int ws_dtype, const void *bias, int bias_dtype, void *y, int y_dtype, int64_t ldy, const float *residual,
                  int64_t ldr, float factor, int64_t m, int64_t n, int64_t k, int flags, void *stream) {
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
    if (y_dtype == KEA_I32) qs = wscale = nullptr;
    const Args a{q, w, ldq, ldw, qs, wscale, bias, y, ldy, residual, ldr, factor, (int)m, (int)n, (int)k,
                 qs_dtype, ws_dtype, bias_dtype, y_dtype, flags};
    // (the tile forms address a tile's rows with 32 bits)
    const int v = ldq < (1 << 23) && ldw < (1 << 23) ? choose(a.m, a.n, a.k) : kSplit32;
    return run(v, a, (hipStream_t)stream);
}

}  // extern "C"
