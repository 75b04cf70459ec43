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
//
// What bounds it: a token reads n k / 2 bytes of weights once (1 x 16384 x 4096: 33.6 MB, 6.5 us at the rate of a large copy; 7.7 us,
// 82 % of it), and below some 8 MB the launch and one walk of k by one workgroup (1 x 2560 x 640 4.7 us; 13 x 1024 x 4096,
// groups of 32, 5.2).
// Many rows are bound by instruction issue: scaling takes eight vector instructions for two products (a conversion and a
// multiply-add for each of four sums), unpacking six for an operand, and little of that hides behind the products of the other wave of a SIMD (4000 x 4096 x 4096: 88 us, 1.5
// POP/s, of 4.1 that the instruction alone reaches here).
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
// registers, U blocks at once, and their sums meet in LDS, added in the waves' order. With 16 columns to a workgroup 1024 outputs
// are 64 of them, whose waves have a few blocks each: a token is two memory round trips.
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

// ---- many rows -----------------------------------------------------------------------------------------------------------------

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

// A workgroup owns BM x BN outputs, WM x WN waves a part each, KG groups of them every KG-th block of 128 k; the groups' sums meet in
// LDS. Stages of such a block for each group stream into LDS by direct copies, NS - 1 ahead: rows of q (unit c of 16 bytes of row r at
// place c ^ r % 8, so that eight rows read together lie in different banks), the weights' tiles and their scales as they are stored.
// A wave unpacks the weights of a stage once for all of its rows; the sums of a block of rows are scaled behind the products of the
// next one. 128 x 128 of eight waves, two workgroups on a CU, are 1.5 POP/s at 4000 x 4096 x 4096; 256 x 256, one on a CU, unpack half as
// much but have nobody to fill the scaling's time (95 us against 88 there), and groups of 32 do not fit their registers. Smaller tiles and
// groups of waves are for outputs that would leave CUs without work.
template <int BM, int BN, int WM, int WN, int KG, int NS, int SCALES, typename ST>
__global__ void __launch_bounds__(WM *WN *KG * 64) tile_kernel(Args p, int tiles_m, int tiles_n) {
    constexpr int NT = WM * WN * 64, RM = BM / WM / 16, RN = BN / WN / 16;
    constexpr int CQ = BM * 8 / NT, CW = BN * 4 / NT, COPIES = CQ + CW;  // copies of a stage by each thread
    constexpr int GROUP = 16 * (int)sizeof(ST), SUNITS = BN / 16 * SCALES * GROUP / 16, SWAVES = (SUNITS + 63) / 64;  // and of the scales by some waves
    static_assert(CQ * NT == BM * 8 && CW * NT == BN * 4 && SUNITS <= NT && NT / 8 % 8 == 0, "copies");
    constexpr int STAGE = BM * 128 + BN * 64 + SWAVES * 1024;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // the group of waves, and within it the thread and wave
    const int kg = __builtin_amdgcn_readfirstlane(threadIdx.x / NT), tid = threadIdx.x % NT, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, i = lane & 15, wm = wave / WN, wn = wave % WN;
    char *const own = lds + kg * NS * STAGE;

    // Workgroups go to the eight XCDs in turn; each XCD takes a run of tiles of its own, in groups of 8 tiles of rows that
    // share their columns, so that what runs at once shares operands in that XCD's L2.
    const int total = tiles_m * tiles_n, per = total / 8, rest = total % 8, x = blockIdx.x % 8;
    const int id = x * per + min(x, rest) + blockIdx.x / 8;
    const int band = id / (8 * tiles_n), in = id % (8 * tiles_n), rows = min(8, tiles_m - 8 * band);
    const int m0 = (8 * band + in % rows) * BM, n0 = in / rows * BN;

    const int last = (p.k - 1) & ~15, last_tile = (p.n + 15) / 16 - 1;
    const int unit = ((tid % 8) ^ (tid / 8 % 8)) * 16;  // of this thread's rows of q, tid / 8 + u NT / 8
    uint32_t q_at[CQ];
#pragma unroll
    for (int u = 0; u < CQ; ++u) q_at[u] = (uint32_t)min(tid / 8 + u * (NT / 8), p.m - 1 - m0) * (uint32_t)p.ldq + unit;
    const int8_t *const q0 = p.q + (long long)m0 * p.ldq;
    const char *w_at[CW];
#pragma unroll
    for (int u = 0; u < CW; ++u) w_at[u] = (const char *)p.words + ((long long)min(n0 / 16 + wave + u * (NT / 64), last_tile) * p.blocks * 64 + lane) * 16;
    // (threads behind the last unit of the scales copy that again)
    const int su = min(tid, SUNITS - 1), s_tile = su / (SCALES * GROUP / 16), s_in = su % (SCALES * GROUP / 16);
    const char *const s_at = (const char *)p.ws + (long long)min(n0 / 16 + s_tile, last_tile) * p.groups * GROUP + s_in % (GROUP / 16) * 16;
    auto copy = [&](int s, int buf) {
        char *const to = own + buf * STAGE;
        const int back = min(0, last - (s * 128 + unit));  // units past the row's end are read from its last one, and meet weights of zero
#pragma unroll
        for (int u = 0; u < CQ; ++u)
            __builtin_amdgcn_global_load_lds((gptr_t)(q0 + s * 128 + (size_t)(q_at[u] + (uint32_t)back)), (lptr_t)(to + (u * NT + wave * 64) * 16), 16, 0, 0);
#pragma unroll
        for (int u = 0; u < CW; ++u)
            __builtin_amdgcn_global_load_lds((gptr_t)(w_at[u] + (long long)s * 1024), (lptr_t)(to + BM * 128 + (u * NT + wave * 64) * 16), 16, 0, 0);
        if (wave >= SWAVES) return;
        const int group = min((s * SCALES + s_in / (GROUP / 16)) >> p.shift, p.groups - 1);
        __builtin_amdgcn_global_load_lds((gptr_t)(s_at + (long long)group * GROUP), (lptr_t)(to + BM * 128 + BN * 64 + wave * 1024), 16, 0, 0);
    };

    v4f acc[RM][RN];
#pragma unroll
    for (int a = 0; a < RM; ++a)
#pragma unroll
        for (int b = 0; b < RN; ++b) acc[a][b] = v4f{0, 0, 0, 0};
    const v4i zero = {0, 0, 0, 0};

#pragma unroll
    for (int s = 0; s < NS - 1; ++s) copy(min(s * KG + kg, p.blocks - 1), s);
    const int i8 = i & 7;
    const uint32_t q_from = (uint32_t)((wm * RM * 16 + i) * 128), w_from = (uint32_t)(BM * 128 + wn * RN * 1024 + lane * 16);
    const uint32_t s_from = (uint32_t)(BM * 128 + BN * 64 + wn * RN * SCALES * GROUP + 4 * g * (int)sizeof(ST));
    int buf = 0;
    for (int s = kg; s < p.blocks + kg; s += KG) {  // (as often for every group)
        // The stage has landed, and every wave has done with the one before, whose buffer takes the copies of the one NS - 1 ahead.
        // (Past the end the last stage is copied again: every stage counts the same copies.)
        if (wave < SWAVES) wait_copies<(NS - 2) * (COPIES + 1)>();
        else wait_copies<(NS - 2) * COPIES>();
        barrier();
        copy(min(s + (NS - 1) * KG, p.blocks - 1), buf ? buf - 1 : NS - 1);
        const char *const from = own + buf * STAGE;
        buf = buf + 1 == NS ? 0 : buf + 1;
        v4i qf[2][2];
        auto fetch = [&](int a) {
#pragma unroll
            for (int h = 0; h < 2; ++h) qf[a & 1][h] = *(const v4i *)(from + q_from + a * 2048 + ((4 * h + g) ^ i8) * 16);
        };
        fetch(0);
        v4i wf[RN][2];
        v4f sf[RN][SCALES];
#pragma unroll
        for (int b = 0; b < RN; ++b) {
            v4i packed = *(const v4i *)(from + w_from + b * 1024);
            if (KG > 1 && s >= p.blocks) packed = zero;  // (a stage past the end)
#pragma unroll
            for (int h = 0; h < 2; ++h) wf[b][h] = weights(packed, h);
#pragma unroll
            for (int c = 0; c < SCALES; ++c) sf[b][c] = scales4((const ST *)(from + s_from + (b * SCALES + c) * GROUP));
        }
        // The products of one block of rows and one group, of all RN tiles, and their scaling, one step behind them.
        v4i sum[2][RN];
        auto products = [&](int step) {
            const int a = step / SCALES, c = step % SCALES;
#pragma unroll
            for (int b = 0; b < RN; ++b) {
                if constexpr (SCALES == 1) {
                    sum[step & 1][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[b][0], qf[a & 1][0], zero, 0, 0, 0);
                } else if constexpr (SCALES == 2) {
                    sum[step & 1][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[b][c], qf[a & 1][c], zero, 0, 0, 0);
                } else {
                    sum[step & 1][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[b][c / 2], g / 2 == c % 2 ? qf[a & 1][c / 2] : zero, zero, 0, 0, 0);
                }
            }
            if constexpr (SCALES == 1)
#pragma unroll
                for (int b = 0; b < RN; ++b) sum[step & 1][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[b][1], qf[a & 1][1], sum[step & 1][b], 0, 0, 0);
        };
        auto scaled = [&](int step) {
            const int a = step / SCALES, c = step % SCALES;
#pragma unroll
            for (int b = 0; b < RN; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[a][b][r] = __builtin_fmaf((float)sum[step & 1][b][r], sf[b][c][r], acc[a][b][r]);
        };
#pragma unroll
        for (int step = 0; step < RM * SCALES; ++step) {
            if (step % SCALES == 0 && step / SCALES + 1 < RM) fetch(step / SCALES + 1);
            products(step);
            if (step) scaled(step - 1);
        }
        scaled(RM * SCALES - 1);
    }
    wait_copies<0>();

    if constexpr (KG > 1) {  // the groups' sums, added in order, by the first
        static_assert(BM * BN * 4 * (KG - 1) <= KG * NS * STAGE, "room for the sums");
        v4f *const part = (v4f *)lds;
        __syncthreads();
        if (kg > 0)
#pragma unroll
            for (int a = 0; a < RM; ++a)
#pragma unroll
                for (int b = 0; b < RN; ++b) part[(((kg - 1) * RM + a) * RN + b) * NT + tid] = acc[a][b];
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int o = 1; o < KG; ++o)
#pragma unroll
            for (int a = 0; a < RM; ++a)
#pragma unroll
                for (int b = 0; b < RN; ++b) acc[a][b] += part[(((o - 1) * RM + a) * RN + b) * NT + tid];
    }
#pragma unroll
    for (int b = 0; b < RN; ++b) {
        const int col = n0 + (wn * RN + b) * 16 + 4 * g;
        if (col >= p.n) continue;
        float bias[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) bias[r] = p.bias ? kea::load_scalar(p.bias, p.bias_dtype, min(col + r, p.n - 1)) : kea::kNoBias;
#pragma unroll
        for (int a = 0; a < RM; ++a) {
            const int row = m0 + (wm * RM + a) * 16 + i;
            if (row < p.m) store4(p, row, col, acc[a][b], kea::load_scalar(p.qs, p.qs_dtype, row), bias);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------

bool scale_type(int t) { return t == KEA_F32 || t == KEA_F16; }
bool aligned(const void *p, int dtype) { return (uintptr_t)p % (dtype == KEA_F32 ? 4 : 2) == 0; }

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_int4_gemm: ") + hipGetErrorString(e));
}

// The form of the shortest estimated time. The figures are fits to what the forms take, hot, as graphs of launches; some of them (us,
// groups of 128 and, behind the stroke, 32; the forms in the order below):
//   4000 x 4096 x 4096   553/718  499/581  468/513  235/358  169/282  131/229   98/201
//   1000 x 4096 x 1024    73/93    36/42    34/38    33/41    24/31    17/23    13/21
//    250 x 4096 x 4096    39/48    34/40    33/37    17/25    13/21    14/22    28/58
//    500 x 1024 x 4096    21/27    19/22    18/20    10/14    12/20    14/21    28/58
//   1000 x 1024 x 1024    21/26    11/13    11/12    10/12     7/9      7/9     12/20
//    375 x 1030 x  641     7/10     5/6      5/6      6/7      7/9      6/8     10/16
//     64 x 1024 x 4096     5/6      7/8     10/13     9/13    12/19    13/21    28/57
// The splitting forms take what one workgroup takes, or what all of them do; the tiles rounds of as many workgroups as run at once,
// with the blocks of 128 k that a group of waves has.
struct Split {
    int rm;
    float one, each, block;  // us: a block of one workgroup alone; of many, every workgroup, and each of its blocks
};
constexpr Split kSplits[] = {{1, 0.075f, 0.0030f, 0.00018f}, {2, 0.128f, 0.0006f, 0.00046f}, {4, 0.244f, 0.0011f, 0.00088f}};
struct Tiles {
    int bm, bn, kg, at_once;
    float base, block, pair;  // us: a launch; a block, with one workgroup on a CU and with two
};
constexpr Tiles kTiles[] = {{32, 64, 4, 256, 4.0f, 0.63f, 0.63f}, {64, 64, 4, 256, 4.9f, 0.95f, 0.95f}, {64, 64, 2, 512, 4.6f, 0.57f, 0.85f}, {128, 128, 1, 512, 5.0f, 0.72f, 1.38f}};

int choose(int m, int n, int blocks, int scales) {
    const float more = scales == 1 ? 1.0f : scales == 2 ? 1.2f : 2.0f, split_more = scales == 1 ? 1.0f : scales == 2 ? 1.06f : 1.25f;
    auto count = [&](int bm, int bn) { return (double)((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
    int best = 0, form = 0;
    double least = 1e30;
    auto take = [&](double t) {
        if (t < least) least = t, best = form;
        ++form;
    };
    for (const Split &f : kSplits) {
        // (rows that are not there are not loaded: 1 x 16384 x 4096 7.8 us, its first form)
        const float used = m < 16 * f.rm ? 0.4f + 0.6f * (float)m / (16 * f.rm) : 1.0f;
        const double one = 2.4 + f.one * blocks * split_more, all = 2.5 + count(16 * f.rm, 16) * (f.each * used + f.block * used * blocks * split_more);
        take(one > all ? one : all);
    }
    for (const Tiles &f : kTiles) {
        const double tiles = count(f.bm, f.bn), rounds = (double)(long long)(tiles / f.at_once), left = tiles - rounds * f.at_once, per = (blocks + f.kg - 1) / f.kg * more;
        const double full = f.pair * per + f.base * 0.6;
        take(f.base * 0.6 + rounds * full + (left > 256 ? full : left > 0 ? f.block * per + f.base * 0.4 : 0.0));
    }
    return best;
}

template <int RM, int SCALES, typename ST, int NW>
int run_split(const Args &a, hipStream_t stream) {
    const int tn = (a.n + 15) / 16;
    const long long tiles = (long long)((a.m + 16 * RM - 1) / (16 * RM)) * tn;
    if (tiles > INT32_MAX / 2 || !kea::fits_dispatch(tiles, NW * 64)) return kea::fail(KEA_EINVAL, "kea_int4_gemm: too large for one launch");
    split_kernel<RM, SCALES, ST, NW, 4 / RM><<<dim3((unsigned)tiles), NW * 64, 0, stream>>>(a, tn);
    return launched();
}

template <int BM, int BN, int WM, int WN, int KG, int NS, int SCALES, typename ST>
int run_tiles(const Args &a, hipStream_t stream) {
    constexpr int NT = WM * WN * KG * 64, lds = KG * NS * (BM * 128 + BN * 64 + (BN / 16 * SCALES * (int)sizeof(ST) + 63) / 64 * 1024);
    static_assert(lds <= 160 * 1024 && NS >= 2, "stage buffers");
    const int tm = (a.m + BM - 1) / BM, tn = (a.n + BN - 1) / BN;
    const long long tiles = (long long)tm * tn;
    if (tiles > INT32_MAX / 2 || !kea::fits_dispatch(tiles, NT)) return kea::fail(KEA_EINVAL, "kea_int4_gemm: too large for one launch");
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)tile_kernel<BM, BN, WM, WN, KG, NS, SCALES, ST>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return kea::fail((int)e, std::string("kea_int4_gemm: ") + hipGetErrorString(e));
    }
    tile_kernel<BM, BN, WM, WN, KG, NS, SCALES, ST><<<dim3((unsigned)tiles), NT, lds, stream>>>(a, tm, tn);
    return launched();
}

template <int SCALES, typename ST>
int run(const Args &a, hipStream_t stream) {
    // (the tile forms address a tile's rows with 32 bits)
    switch (a.ldq < (1 << 23) ? choose(a.m, a.n, a.blocks, SCALES) : 2) {
        // (eight waves where four would load their blocks of k in more than one turn, and no more than two workgroups meet on a CU: 1 x
        // 1024 x 16384 6.2 us and 7.3 with four, 13 x 1024 x 4096 5.2 and 5.5 from cold weights; 1 x 4096 x 1024 3.2 and 2.7, 1 x 16384 x
        // 4096 8.0 and 7.6 from cold weights)
        case 0: return a.blocks > 16 && (long long)((a.m + 15) / 16) * ((a.n + 15) / 16) <= 512 ? run_split<1, SCALES, ST, 8>(a, stream) : run_split<1, SCALES, ST, 4>(a, stream);
        case 1: return run_split<2, SCALES, ST, 4>(a, stream);
        case 2: return run_split<4, SCALES, ST, 4>(a, stream);
        case 3: return run_tiles<32, 64, 1, 4, 4, 3, SCALES, ST>(a, stream);
        case 4: return run_tiles<64, 64, 2, 2, 4, 2, SCALES, ST>(a, stream);
        case 5: return run_tiles<64, 64, 2, 2, 2, 3, SCALES, ST>(a, stream);
        default: return run_tiles<128, 128, 2, 4, 1, 2, SCALES, ST>(a, stream);
    }
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
