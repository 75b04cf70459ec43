// Attention within a sliding window and to the first tokens (include/kea_block.h).
//
// The query heads that share a key head are rows of one problem: row r of a sequence and key head is query r / group, head
// r % group of the group, so that a tile of rows stands at few positions and their keys are read once. A workgroup takes
// 32 WQ rows and walks the keys that any of them sees, first those of the first tokens that lie before the window, then the
// window, in tiles that it copies straight to LDS one ahead. Per tile and wave:
//   S^T = K Q^T        keys are the matrix instruction's rows, queries its columns: a lane holds 16 keys' scores of one
//                      query (its column), and the maximum over keys is 15 steps in the lane and one across its halves
//   p = 2^(s - m)      base 2 with the scale folded into one fma; the reference m is raised, and the sums rescaled, only
//                      when a score passes it by more than 8, so most tiles leave the output's accumulators alone
//   O^T += V^T P^T     the scores' layout is the second operand's of this product up to the order of keys, which the sum does
//                      not depend on: V's columns are read in that order (ds_read_b64_tr_b16, which transposes on the way;
//                      single words for FP32), and probabilities never leave the registers
// WQ waves share out the rows (many queries), or WK waves the keys of each tile (few queries), whose parts meet in LDS. Where
// that still leaves few workgroups the keys are split over several, whose parts a second launch joins.
//
// Measured (heads of 128, BF16, 8 on 4, causal): 32768 tokens with a window of 1023 174 us, 790 TFLOP/s of the pairs that are
// seen (a large product reaches 1250); 10000 of them 70 to 78 us, in two rounds of workgroups of which the second fills a
// quarter of the chip. Matrix instructions take half of such a wave's time: its softmax and the LDS reads are in line with
// them, two waves a SIMD overlap in part, and the clock falls to 1.9 GHz. FP32: the matrix instruction (73 % of a tile's
// cycles). One token of 16 sequences against 1028 keys each: 13.2 us in two launches, latency of 64 KB a CU and of the join.
//
// Keys outside the tile's range are read from its last key and masked. A masked score is -infinity whatever K holds, but a
// product with its weight of 0 is NaN where V is infinite or NaN. Such a sum shows in the output: a workgroup that ends up
// with a value that is not finite does its work a second time with those elements of V taken out of the product and added to
// the queries that see them, and (FP32 and BF16) a third time for rows that are still not finite, with values of 2^-40 of their
// size, whose sums are finite. (In such rows, and there alone, elements of values below 2^-86 lose digits.) A row's bits depend on
// the keys that it sees alone: its maximum, sums and passes are decided by its own scores and sums.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "kea_internal.h"
#include "../../include/kea_block.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void *lptr_t;
typedef __attribute__((address_space(3))) v4s *ltr_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;  // scores may pass the reference by this much (base 2) before it is raised

// The exponent e with 2^(e - 1) <= v < 2^e; 0 for 0, infinities and NaN.
__device__ __forceinline__ int exponent(float v) { return __builtin_amdgcn_frexp_expf(v); }

struct Args {
    kea_heads q, k, v, out;
    const int32_t *lengths, *starts;
    float *part, *stats;  // splits > 1: [splits][sequences and key heads][rows][d], [..][rows][2] (see join_kernel)
    int batch, tq, tk, kv_heads, group, d, left, right, sinks;
    int rows, row_tiles, splits;
    int by_group;  // the grid is [sequences and key heads][tiles][splits], or [tiles][sequences and key heads][splits]
    uint32_t group_mul, group_shift, heads_mul, heads_shift;
    float scale;

    // row / group and (sequence and key head) / kv_heads, for numbers below 2^31: mul = 2^(31 + s) / divisor + 1 with
    // 2^s >= divisor
    __device__ __forceinline__ int token(int row) const { return (int)(__umulhi(2u * (uint32_t)row, group_mul) >> group_shift); }
    __device__ __forceinline__ int sequence(int bh) const { return (int)(__umulhi(2u * (uint32_t)bh, heads_mul) >> heads_shift); }
};

template <int N>
struct Count {
    static constexpr int value = N;
};

template <typename T, int DP, int WQ, int WK>
struct Shape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int NW = WQ * WK, NT = 64 * NW;
    // 32-key blocks of a tile: the waves' one each where they share out the keys, otherwise what 32 KB hold, two at most
    static constexpr int KB = WK > 1 ? WK : (2 * 2 * 32 * DP * (int)sizeof(T) <= 32768 ? 2 : 1);
    static constexpr int NB = KB / WK, KT = 32 * KB;
    static constexpr int ROW = DP * (int)sizeof(T), UNITS = ROW / 16, BUF = 2 * KT * ROW;
    static constexpr int MERGE = WK > 1 ? NW * 32 * (DP + 2) * 4 : 0;
    // two buffers where two workgroups of a CU have room for them, otherwise one: the other workgroup works meanwhile
    static constexpr int BUFFERS = 2 * BUF <= 65536 ? 2 : 1;
    static constexpr int LDS = (BUFFERS * BUF > MERGE ? BUFFERS * BUF : MERGE) + 64;
};

// The place of 16-byte unit c of a key's row in LDS is c ^ swizzle(key), so that rows read together lie in different banks.
// K: eight (16) rows at one unit. V of 16-bit types: four rows at two neighbouring pairs of units, which stay pairs. Either
// depends on key % 32 alone.
template <bool F32, int UNITS>
__device__ __forceinline__ int swizzle_k(int key) {
    return F32 ? key & 7 : UNITS == 8 ? key >> 1 & 7 : key & 15;
}
template <bool F32, int UNITS>
__device__ __forceinline__ int swizzle_v(int key) {
    return F32 ? key & 7 : UNITS == 8 ? (key >> 1 & 1) * 4 : (key & 3) * 4;
}

// A lane's value and that of the lane 32 away, the lower half's first. (The components are read before they are cast:
// hipcc's __builtin_bit_cast of a component access gives component 0.)
__device__ __forceinline__ float2 halves(float v) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t lower = s[0], upper = s[1];
    return make_float2(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper));
}
__device__ __forceinline__ float other_half_max(float v) {
    const float2 s = halves(v);
    return fmaxf(s.x, s.y);
}
__device__ __forceinline__ float both_halves(float v) {
    const float2 s = halves(v);
    return s.x + s.y;
}

// 16 bytes a lane from global memory straight to LDS, at the wave's base address plus 16 a lane; done when vmcnt says so. In
// place of the builtin, after which the compiler waits for all of a wave's copies before its next transposing read, those for
// the tile ahead among them. (Nothing else here uses m0.) The second form reads at a uniform address plus an offset.
__device__ __forceinline__ void copy16(const void *src, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(src) : "memory");
}
__device__ __forceinline__ void copy16(const void *src, uint32_t offset, uint32_t base) {
    const uint64_t at = (uint64_t)(uintptr_t)src;
    const uint64_t uniform = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(offset), "s"(uniform) : "memory");
}

template <typename T>
__device__ __forceinline__ v16f mma(v8s a, v8s b, v16f c) {
    if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// c + the two weights of a pair: FP32, to 2.7 u of it (measured), where two additions would be off by 2 u. (T: the pair's type.)
template <typename T>
__device__ __forceinline__ float add_pair(const T *w, float c) {
    typedef T pair __attribute__((ext_vector_type(2)));
    const pair ones = {(T)1.0f, (T)1.0f};
    if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_fdot2(*(const pair *)w, ones, c, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(*(const pair *)w, ones, c, false);
}

__device__ __forceinline__ bool finite(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) != 0x7F800000u; }
// Whether an element of 16 or 32 bits is an infinity or NaN, and a unit of eight or four without such elements.
template <typename T>
__device__ __forceinline__ bool finite_bits(T v) {
    return finite((float)v);
}

// RAGGED: d < DP, rows of K and V end before DP elements and go through registers, zeros behind them.
template <typename T, int DP, int WQ, int WK, bool RAGGED>
__global__ void __launch_bounds__(64 * WQ *WK, DP *sizeof(T) <= 256 ? 2 : 1) window_kernel(Args a) {
    using S = Shape<T, DP, WQ, WK>;
    constexpr bool F32 = S::F32;
    constexpr int NB = S::NB, KT = S::KT, UNITS = S::UNITS, NT = S::NT, ROW = S::ROW, EPU = 16 / (int)sizeof(T);
    constexpr int QF = DP / 16, DB = DP / 32;  // steps of 16 elements, blocks of 32 output elements
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t *const flags = (uint32_t *)(lds + S::LDS - 64);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5, wq = wave / WK, wk = wave % WK;

    // Workgroups go to the eight XCDs in turn, and the first grid dimension is a multiple of eight (or alone on its row): with
    // eight sequences and key heads or more, one XCD takes all tiles of each of them; otherwise runs of neighbouring tiles.
    // Either way what shares keys shares an L2. (Of the last up to seven workgroups of a row some have nothing to do.)
    int tile, bh;
    if (a.by_group) {
        bh = blockIdx.x, tile = blockIdx.y;
    } else {
        const int x = blockIdx.x, run = (int)gridDim.x / 8;
        bh = blockIdx.y, tile = run ? x % 8 * run + x / 8 : x;
    }
    if (bh >= a.batch * a.kv_heads || tile >= a.row_tiles) return;
    const int split = blockIdx.z, b = a.sequence(bh), hk = bh - b * a.kv_heads;
    // (uniform, which the compiler does not see of loaded values)
    const int len = __builtin_amdgcn_readfirstlane(a.lengths ? min(max(a.lengths[b], 0), a.tk) : a.tk);
    const int start = __builtin_amdgcn_readfirstlane(a.starts ? min(max(a.starts[b], -(1 << 30)), 1 << 30) : len - a.tq);

    // this lane's query
    const int r0 = tile * 32 * WQ, row = r0 + 32 * wq + n;
    const bool real = row < a.rows;
    const int t = a.token(min(row, a.rows - 1)), head = hk * a.group + min(row, a.rows - 1) - t * a.group, p = start + t;
    const bool inside = real && p >= 0 && p < len;
    // positions of the tile's and of the wave's rows, those inside the sequence
    auto first_of = [&](int from) { return max(start + a.token(min(from, a.rows - 1)), 0); };
    auto last_of = [&](int from, int rows) { return min(start + a.token(min(from + rows, a.rows) - 1), len - 1); };
    auto reach = [&](int from) { return (int)min((long long)len - 1, (long long)from + a.right); };  // the last key seen from there
    const int p0 = first_of(r0), p1 = last_of(r0, 32 * WQ);
    const int w0 = first_of(r0 + 32 * wq), w1 = r0 + 32 * wq < a.rows ? last_of(r0 + 32 * wq, 32) : -1;

    // The keys that some row of the tile sees, numbered on: v < first is key v, others key v + shift.
    int low = max(0, p0 - a.left), first = min(a.sinks, low), keys = 0;
    if (first == low) first = low = 0;
    const int shift = low - first, sinks = shift ? first : a.sinks;
    if (p0 <= p1) keys = reach(p1) + 1 - shift;
    int from = 0, to = keys;
    if (a.splits > 1) {
        const int share = ((keys + 31) / 32 + a.splits - 1) / a.splits * 32;
        from = min(keys, split * share);
        to = min(keys, from + share);
    }
    const int tiles = (to - from + KT - 1) / KT;
    // per lane and wave, in these numbers: the last key seen and the first of the window
    const int hi = reach(max(p, 0)) - shift, lo = max(p, 0) - a.left - shift;
    const int hi0 = reach(w0) - shift, hi1 = reach(w1) - shift, lo0 = w0 - a.left - shift, lo1 = w1 - a.left - shift;

    const T *const kp = (const T *)a.k.data_dev + b * a.k.batch_stride + hk * a.k.head_stride;
    const T *const vp = (const T *)a.v.data_dev + b * a.v.batch_stride + hk * a.v.head_stride;
    // the copies of this thread: unit tid + u NT of a tile of K and of V, rows STEP apart at one place
    constexpr int STEP = NT / UNITS, COPIES = KT / STEP;
    static_assert(NT % UNITS == 0 && (STEP % 16 == 0 || STEP == 8 || STEP == 4 || STEP == 2 || STEP == 1), "copies");
    const int key0 = tid / UNITS;
    auto unit = [&](int kv, int key) { return (tid % UNITS ^ (kv ? swizzle_v<F32, UNITS>(key) : swizzle_k<F32, UNITS>(key))) * EPU; };
    // a tile of neighbouring keys is copied from a uniform address, each thread's rows at 32-bit offsets from it, where those
    // suffice: as many offsets as the swizzle has values over the thread's rows
    constexpr int PERIOD = F32 ? 8 : 16, OFFSETS = STEP < PERIOD ? PERIOD / STEP : 1;
    constexpr bool NEAR = !RAGGED && OFFSETS <= 4;
    const bool near_k = (long long)KT * a.k.t_stride < 1 << 29, near_v = (long long)KT * a.v.t_stride < 1 << 29;
    uint32_t off_k[OFFSETS], off_v[OFFSETS];
#pragma unroll
    for (int u = 0; u < OFFSETS; ++u) {
        off_k[u] = ((uint32_t)key0 * (uint32_t)a.k.t_stride + unit(0, key0 + u * STEP)) * (uint32_t)sizeof(T);
        off_v[u] = ((uint32_t)key0 * (uint32_t)a.v.t_stride + unit(1, key0 + u * STEP)) * (uint32_t)sizeof(T);
    }
    auto stage = [&](int v0, int buf, bool of_k, bool of_v) {
        // (made anew on every call: kept for all copies of a tile, the addresses would not fit the registers)
        uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)lds + buf * S::BUF + wave * 1024);
        int v1 = __builtin_amdgcn_readfirstlane(v0);
        asm volatile("" : "+s"(dst), "+s"(v1));
        if (NEAR && near_k && near_v && v1 >= first && v1 + KT <= to) {
            auto copy = [&](const T *from, long long stride, const uint32_t (&offset)[OFFSETS], uint32_t at) {
                from += (long long)(v1 + shift) * stride;
#pragma unroll
                for (int u = 0; u < COPIES; ++u) {
                    copy16(from, offset[u % OFFSETS], at);
                    from += STEP * stride;
                    at += NT * 16;
                }
            };
            if (of_k) copy(kp, a.k.t_stride, off_k, dst);
            if (of_v) copy(vp, a.v.t_stride, off_v, dst + KT * ROW);
            return;
        }
        auto copy = [&](const T *from, long long stride, int kv, uint32_t at) {
#pragma unroll
            for (int u = 0; u < COPIES; ++u) {
                const int key = key0 + u * STEP, v = min(v1 + key, to - 1), c = unit(kv, key);
                const T *src = from + (long long)(v + (v >= first ? shift : 0)) * stride + c;
                if constexpr (RAGGED) {
                    const v4f zero = {0, 0, 0, 0};
                    *(v4f *)(lds + buf * S::BUF + kv * KT * ROW + (u * NT + tid) * 16) = c < a.d ? *(const v4f *)src : zero;
                } else {
                    copy16(src, at);
                    at += NT * 16;
                }
            }
        };
        if (of_k) copy(kp, a.k.t_stride, 0, dst);
        if (of_v) copy(vp, a.v.t_stride, 1, dst + KT * ROW);
    };
    // All but the last LEFT of this wave's copies have landed and its LDS reads are done; then all waves'.
    auto landed = [&](auto left) {
        constexpr int LEFT = RAGGED ? 0 : decltype(left)::value;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((LEFT & 15) | ((LEFT >> 4) << 14) | (7 << 4));  // vmcnt(LEFT) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // the query as the product's second operand: elements 16 c + 8 h .. of its row (FP32: 8 c + 4 h ..)
    v8s qf[F32 ? 1 : QF];
    v4f qx[F32 ? 2 * QF : 1];
    {
        const T *qp = (const T *)a.q.data_dev + b * a.q.batch_stride + (long long)t * a.q.t_stride + head * a.q.head_stride;
        if constexpr (F32) {
#pragma unroll
            for (int c = 0; c < 2 * QF; ++c) qx[c] = v4f{0, 0, 0, 0};
            if (inside)
#pragma unroll
                for (int c = 0; c < 2 * QF; ++c)
                    if (!RAGGED || 8 * c + 4 * h < a.d) qx[c] = *(const v4f *)(qp + 8 * c + 4 * h);
            if (a.scale < 0)
#pragma unroll
                for (int c = 0; c < 2 * QF; ++c) qx[c] = -qx[c];
            if (a.scale == 0)
#pragma unroll
                for (int c = 0; c < 2 * QF; ++c) qx[c] *= 0.0f;
        } else {
#pragma unroll
            for (int c = 0; c < QF; ++c) qf[c] = v8s{0, 0, 0, 0, 0, 0, 0, 0};
            if (inside)
#pragma unroll
                for (int c = 0; c < QF; ++c)
                    if (!RAGGED || 16 * c + 8 * h < a.d) qf[c] = *(const v8s *)(qp + 16 * c + 8 * h);
            if (a.scale < 0)
#pragma unroll
                for (int c = 0; c < QF; ++c) qf[c] ^= (short)0x8000;
            if (a.scale == 0)
#pragma unroll
                for (int c = 0; c < QF; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) qf[c][e] = __builtin_bit_cast(short, (T)((float)__builtin_bit_cast(T, (short)qf[c][e]) * 0.0f));
        }
    }
    // (a scale of 0 would make a masked score's -infinity NaN: it is in the queries then)
    const float scale = a.scale != 0 ? fabsf(a.scale) * kLog2e : 1.0f;

    v16f o[DB];
    float m = -INFINITY, l = 0.0f;  // l: this half's keys
    int pass = 0;
    uint32_t small = 0;  // the wave's rows that the third pass is for
    constexpr int kDown = 40;  // 2^30 keys of weights up to 2^8

    // operand addresses in a tile, as offsets: K unit 2 c + h of row n is at ka ^ 32 c, V units 4 d .. of its rows at va ^ 64 d
    // (FP32: word n of units 8 d .. at va ^ 128 d)
    int ka = n * ROW + (h ^ swizzle_k<F32, UNITS>(n)) * 16 + 32 * wk * ROW;
    int va;
    if constexpr (F32) {
        va = 4 * h * ROW + n % 4 * 4 + 32 * wk * ROW;
    } else {
        const int key = 4 * h + (lane & 15) / 4;
        va = key * ROW + ((2 * (lane >> 4 & 1) + (lane & 3) / 2) ^ swizzle_v<F32, UNITS>(key)) * 16 + (lane & 1) * 8 + 32 * wk * ROW;
    }

    // a tile that none of the wave's rows sees (the whole of it lies outside their windows)
    auto unseen = [&](int v0) { return w0 > w1 || v0 > hi1 || (v0 + KT <= lo0 && v0 >= sinks); };
    v16f s[NB];
    auto scores = [&](int v0, int buf) {
        if (unseen(v0)) return;
        const char *const kt = lds + buf * S::BUF;
        asm volatile("" : "+v"(ka));  // (the addresses made from it are made anew, not kept for every use; va likewise)
        // Operands are read a step ahead of the matrix instructions that take them, into one of two register sets.
        constexpr int KSTEPS = F32 ? 2 * QF : QF / 2;  // steps of eight elements (FP32) or 32
#pragma unroll
        for (int i = 0; i < NB; ++i) s[i] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        v4f kx[2][NB][F32 ? 1 : 2];
        auto read_k = [&](int c) {
#pragma unroll
            for (int y = 0; y < (F32 ? 1 : 2); ++y)
#pragma unroll
                for (int i = 0; i < NB; ++i) kx[c & 1][i][y] = *(const v4f *)(kt + (ka ^ 32 * (F32 ? c : 2 * c + y)) + 32 * i * WK * ROW);
        };
        read_k(0);
#pragma unroll
        for (int c = 0; c < KSTEPS; ++c) {
            if (c + 1 < KSTEPS) read_k(c + 1);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < NB; ++i) s[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(kx[c & 1][i][0][e], qx[c][e], s[i], 0, 0, 0);
            } else {
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < NB; ++i) s[i] = mma<T>(__builtin_bit_cast(v8s, kx[c & 1][i][y]), qf[2 * c + y], s[i]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto output = [&](int v0, int buf) {
        if (unseen(v0)) return;
        const char *const vt = lds + buf * S::BUF + KT * ROW;
        asm volatile("" : "+v"(va));
        // V: steps of one key of each half (FP32) or 16 keys, the first read while the softmax runs
        constexpr int VSTEPS = NB * (F32 ? 16 : 2);
        float vx[2][F32 ? DB : 1];
        v4s vh[2][F32 ? 1 : DB][2];
        auto read_v = [&](int j) {
            if constexpr (F32) {
                // V[8 (e / 4) + e % 4 + 4 h][32 d + n]: unit 8 d + n / 4 at its place
                const int i = j / 16, key = 8 * (j % 16 / 4) + j % 4;
                const char *const at = vt + va + (32 * i * WK + key) * ROW + ((n / 4) ^ ((key + 4 * h) & 7)) * 16;
#pragma unroll
                for (int d = 0; d < DB; ++d) vx[j & 1][d] = *(const float *)(at + 128 * d);
            } else {
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const char *const at = vt + (va ^ 64 * d) + (32 * (j / 2) * WK + 16 * (j % 2)) * ROW;
                    vh[j & 1][d][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ltr_t)at);
                    vh[j & 1][d][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ltr_t)(at + 8 * ROW));
                }
            }
        };
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
        // masks, where the tile is not seen as a whole by every row of the wave
        const bool whole = v0 + KT <= to && v0 + KT - 1 <= hi0 && (v0 >= lo1 || v0 + KT <= sinks);
        if (!whole) {
            const int off = v0 + 32 * wk + 4 * h, hx = min(to - 1, hi) - off, lx = max(lo, v0 - KT) - off, sx = min(sinks, v0 + KT) - off;
            const uint32_t width = (uint32_t)max(hx - lx + 1, 0);
            if (v0 >= sinks) {
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if ((uint32_t)(32 * i * WK + 8 * (e / 4) + e % 4 - lx) >= width) s[i][e] = -INFINITY;
            } else {
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int at = 32 * i * WK + 8 * (e / 4) + e % 4;
                        if (!(at <= hx && (at >= lx || at < sx))) s[i][e] = -INFINITY;
                    }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[i][e]);
        top = other_half_max(top) * scale;
        if (__any(top > m + kLazy)) {
            const float next = top > m + kLazy ? top : m;
            if (__any(m != -INFINITY)) {  // (nothing is there to rescale at first)
                const float by = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
                l *= by;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] *= by;
            }
            m = next;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[i][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], scale, -ref));
                if constexpr (F32) sum += s[i][e];
            }
        // The 16-bit types' weights are rounded to what the product takes (half a step, relative to themselves; below the
        // smallest normal FP16 number 2^-25): as accurate as the values they weigh, and the error of the output, relative to it,
        // is 0.0021 in BF16 where its own rounding alone gives 0.0016. (Weights in two parts would double this product's matrix
        // instructions, half of all.) Their sum is of the rounded ones, so that they add up to one and the output stays among the
        // values.
#pragma unroll
        for (int j = 0; j < VSTEPS; ++j) {
            if (j + 1 < VSTEPS) read_v(j + 1);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (F32) {
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vx[j & 1][d], s[j / 16][j % 16], o[d], 0, 0, 0);
            } else {
                T w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = (T)s[j / 2][8 * (j % 2) + e];
#pragma unroll
                for (int e = 0; e < 8; e += 2) sum = add_pair<T>(w + e, sum);
                const v8s pf = *(const v8s *)w;
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const v4s x0 = vh[j & 1][d][0], x1 = vh[j & 1][d][1];
                    o[d] = mma<T>(v8s{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]}, pf, o[d]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum;
        if (__builtin_expect(pass > 0, 0)) {
            for (int i = 0; i < NB; ++i) {
                uint32_t left = __builtin_amdgcn_readfirstlane(flags[i * WK + wk]);
                while (left) {
                    const int v = v0 + 32 * (i * WK + wk) + __builtin_ctz(left);
                    left &= left - 1;
                    if (!(v <= min(to - 1, hi) && (v >= lo || v < sinks))) continue;
                    const T *src = vp + (long long)(v + (v >= first ? shift : 0)) * a.v.t_stride;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
                        for (int e = 0; e < 16; ++e) {
                            const int at = 32 * d + 8 * (e / 4) + 4 * h + e % 4;
                            if (at < a.d && !finite_bits(src[at])) o[d][e] += (float)src[at];
                        }
                }
            }
        }
    };
    // V's elements that are no numbers become zeros in LDS, and their keys' flags are set; in the third pass the others are scaled.
    auto take_out = [&](int buf) {
        const float by = pass == 2 ? __builtin_amdgcn_ldexpf(1.0f, -kDown) : 1.0f;
        if (tid < S::KB) flags[tid] = 0;
        __syncthreads();
        for (int at = tid; at < KT * UNITS; at += NT) {
            T *unit = (T *)(lds + buf * S::BUF + KT * ROW + at * 16);
            bool any = false;
            for (int e = 0; e < EPU; ++e) {
                if (!finite_bits(unit[e])) unit[e] = (T)0.0f, any = true;
                else if (pass == 2) unit[e] = (T)((float)unit[e] * by);
            }
            if (any) atomicOr(&flags[at / UNITS / 32], 1u << (at / UNITS % 32));
        }
        __syncthreads();
    };

    constexpr int PER = WK > 1 ? 32 * (DP / 4) / NT : 1;  // units of four outputs that each thread joins
    const int rows = min(32 * WQ, a.rows - r0);
    v4f joined[PER];
    float2 refs[PER];
    const long long slot0 = ((long long)split * a.batch * a.kv_heads + bh) * a.rows;
    T *const out = (T *)a.out.data_dev + b * a.out.batch_stride;
    // Stores the rows of `done`, whose sums are 2^-up of their size.
    auto store = [&](uint32_t done, int up) {
        // (addresses made here, not kept through the passes for both calls)
        int thread = tid, of = row;
        asm volatile("" : "+v"(thread), "+v"(of));
        if constexpr (WK == 1) {
            if (real && (done >> n & 1)) {
                if (a.splits > 1) {
                    float *const part = a.part + (slot0 + of) * a.d;
                    const float unit = __builtin_amdgcn_ldexpf(1.0f, up - exponent(l));
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            if (!RAGGED || 32 * d + 2 * e + 4 * h < a.d) *(v4f *)(part + 32 * d + 2 * e + 4 * h) = v4f{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]} * unit;
                    if (h == 0) *(float2 *)(a.stats + 2 * (slot0 + of)) = make_float2(m, l);
                } else {
                    T *const y = out + (long long)t * a.out.t_stride + head * a.out.head_stride + 4 * h;
                    const float by = l != 0.0f ? __builtin_amdgcn_ldexpf(1.0f / l, up) : 0.0f;
                    const bool some = inside && l != 0.0f;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            if (RAGGED && 32 * d + 2 * e + 4 * h >= a.d) continue;
                            T v[4];
#pragma unroll
                            for (int z = 0; z < 4; ++z) v[z] = (T)(some ? o[d][e + z] * by : 0.0f);
                            if constexpr (F32) *(v4f *)(y + 32 * d + 2 * e) = *(const v4f *)v;
                            else *(v4s *)(y + 32 * d + 2 * e) = *(const v4s *)v;
                        }
                }
            }
        } else {
            static_assert(WQ == 1, "one group of rows");
#pragma unroll
            for (int u = 0; u < PER; ++u) {
                const int at = u * NT + thread, r = at / (DP / 4), c = at % (DP / 4);
                if (r >= rows || (RAGGED && 4 * c >= a.d) || !(done >> r & 1)) continue;
                if (a.splits > 1) {
                    *(v4f *)(a.part + (slot0 + r0 + r) * a.d + 4 * c) = joined[u] * __builtin_amdgcn_ldexpf(1.0f, up - exponent(refs[u].y));
                    if (c == 0) *(float2 *)(a.stats + 2 * (slot0 + r0 + r)) = refs[u];
                    continue;
                }
                const int tt = a.token(r0 + r), pp = start + tt;
                const bool some = pp >= 0 && pp < len && refs[u].y != 0.0f;
                const float by = __builtin_amdgcn_ldexpf(1.0f / refs[u].y, up);
                T *const y = out + (long long)tt * a.out.t_stride + (hk * a.group + r0 + r - tt * a.group) * a.out.head_stride + 4 * c;
                T res[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) res[e] = (T)(some ? joined[u][e] * by : 0.0f);
                if constexpr (F32) *(v4f *)y = *(const v4f *)res;
                else *(v4s *)y = *(const v4s *)res;
            }
        }
    };
    for (;; ++pass) {
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        m = -INFINITY;
        l = 0.0f;
        if (tiles) stage(from, 0, true, true);
        if constexpr (S::BUFFERS == 2) {
            for (int i = 0; i < tiles; ++i) {
                const int v0 = from + i * KT, buf = i & 1;
                landed(Count<0>());
                if (pass) take_out(buf);
                if (i + 1 < tiles) stage(v0 + KT, buf ^ 1, true, true);
                scores(v0, buf);
                output(v0, buf);
            }
        } else {
            // one buffer of K and one of V: a tile's V is on its way during its scores, the next tile's K during its outputs
            for (int i = 0; i < tiles; ++i) {
                const int v0 = from + i * KT;
                if (i == 0) landed(Count<COPIES>());
                else landed(Count<0>());
                if (i) stage(v0, 0, false, true);
                scores(v0, 0);
                landed(Count<0>());
                if (i + 1 < tiles) stage(v0 + KT, 0, true, false);
                if (pass) take_out(0);
                output(v0, 0);
            }
        }
        l = both_halves(l);
        bool bad = false;
        uint32_t bad_rows = 0;
        if constexpr (WK == 1) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                float z = 0.0f;  // (an infinity or NaN times 0 is NaN)
#pragma unroll
                for (int e = 0; e < 16; ++e) z = __builtin_fmaf(o[d][e], 0.0f, z);
                bad |= z != z;
            }
        } else {
            // the waves' parts of each row meet in LDS: [wave][32][DP] outputs, then [wave][32][2] maxima and sums
            float *const po = (float *)lds, *const ps = po + S::NW * 32 * DP;
            __syncthreads();
            if (n < rows) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        // (units of four elements, swizzled by the row: 32 rows are written at once)
                        const int c = 8 * d + e / 2 + h;
                        *(v4f *)(po + ((wave * 32 + n) * (DP / 4) + (c ^ (n & 7))) * 4) = v4f{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
                    }
                if (h == 0) *(float2 *)(ps + 2 * (wave * 32 + n)) = make_float2(m, l);
            }
            __syncthreads();
            // (a wave that saw nothing of a row has zeros there and weighs nothing; rows past the last are the last again)
            float2 part[PER][WK];
            v4f share[PER][WK];
#pragma unroll
            for (int u = 0; u < PER; ++u) {
                const int at = u * NT + tid, r = min(at / (DP / 4), rows - 1), c = at % (DP / 4);
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    part[u][w] = *(const float2 *)(ps + 2 * (w * 32 + r));
                    share[u][w] = *(const v4f *)(po + ((w * 32 + r) * (DP / 4) + (c ^ (r & 7))) * 4);
                }
            }
#pragma unroll
            for (int u = 0; u < PER; ++u) {
                float top = part[u][0].x, all = 0.0f;
#pragma unroll
                for (int w = 1; w < WK; ++w) top = fmaxf(top, part[u][w].x);
                v4f v = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    const float by = part[u][w].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(part[u][w].x - top);
                    all += part[u][w].y * by;
                    v += share[u][w] * by;
                }
                joined[u] = v;
                refs[u] = make_float2(top, all);
                const float z = (v[0] * 0.0f + v[1] * 0.0f) + (v[2] * 0.0f + v[3] * 0.0f);  // (an infinity or NaN times 0 is NaN)
                if (z != z) bad = true, bad_rows |= 1u << min((u * NT + tid) / (DP / 4), rows - 1);
            }
        }
        if (pass == (__is_same(T, _Float16) ? 1 : 2) || !__syncthreads_or(bad)) break;
        if (__builtin_expect(pass == 1, 0)) {
            if constexpr (WK == 1) {
                const uint64_t lanes = __ballot(bad);
                small = (uint32_t)lanes | (uint32_t)(lanes >> 32);
            } else {
                if (tid == 0) flags[8] = 0;
                __syncthreads();
                if (bad_rows) atomicOr(&flags[8], bad_rows);
                __syncthreads();
                small = __builtin_amdgcn_readfirstlane(flags[8]);
            }
            store(~small, 0);
        }
    }
    store(pass == 2 ? small : ~0u, pass == 2 ? kDown : 0);
}

// Joins the splits: out = sum_s O_s 2^(m_s - m) / sum_s l_s 2^(m_s - m), four elements a thread, eight splits at a time. The parts
// hold O_s 2^-e_s and the sum so far is kept at 2^-e of its size, e_s and e the exponents of l_s and of the sum of weights: that is
// below the largest value and a half or more of the weighted mean, so it neither overflows nor loses digits that the mean has.
template <typename T>
__global__ void __launch_bounds__(64) join_kernel(Args a) {
    const int at = blockIdx.x * 64 + threadIdx.x, per = a.d / 4, r = at / per, c = at - r * per, bh = blockIdx.y, b = a.sequence(bh), hk = bh - b * a.kv_heads;
    if (r >= a.rows) return;
    const int row = bh * a.rows + r, all = a.batch * a.kv_heads * a.rows, t = a.token(r);
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.tk) : a.tk;
    const int p = (a.starts ? min(max(a.starts[b], -(1 << 30)), 1 << 30) : len - a.tq) + t;
    float m = -INFINITY, sum = 0.0f;
    int e = 0;
    v4f v = {0, 0, 0, 0};
    for (int s0 = 0; s0 < a.splits; s0 += 8) {
        float2 stat[8];
        v4f part[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const long long slot = (long long)min(s0 + s, a.splits - 1) * all + row;
            stat[s] = *(const float2 *)(a.stats + 2 * slot);
            part[s] = *(const v4f *)(a.part + slot * a.d + 4 * c);
        }
        float top = m;
#pragma unroll
        for (int s = 0; s < 8; ++s) top = s0 + s < a.splits ? fmaxf(top, stat[s].x) : top;
        const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        sum *= old;
        float by[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            by[s] = stat[s].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(stat[s].x - top);  // (a NaN stays one)
            if (s0 + s < a.splits) sum += stat[s].y * by[s];
        }
        const int next = exponent(sum);
        v *= __builtin_amdgcn_ldexpf(old, e - next);
        e = next;
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s0 + s < a.splits) v += part[s] * __builtin_amdgcn_ldexpf(by[s], exponent(stat[s].y) - e);
    }
    const float by = p >= 0 && p < len && sum != 0.0f ? __builtin_amdgcn_ldexpf(1.0f / sum, e) : 0.0f;
    T res[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) res[i] = (T)(by == 0.0f ? 0.0f : v[i] * by);
    T *const y = (T *)a.out.data_dev + b * a.out.batch_stride + (long long)t * a.out.t_stride + (hk * a.group + r - t * a.group) * a.out.head_stride + 4 * c;
    if constexpr (sizeof(T) == 4) *(v4f *)y = *(const v4f *)res;
    else *(v4s *)y = *(const v4s *)res;
}

// ---- host ----------------------------------------------------------------------------------------------------------------------

struct Plan {
    bool few;            // waves share out the keys of 32 rows, not the rows
    int dp, row_tiles, splits;
    int64_t rows, part_bytes, stats_bytes;
};

int plan_of(int dtype, int64_t batch, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d, int64_t left, int64_t right,
            int64_t sinks, Plan *out) {
    Plan p{};
    p.dp = d <= 64 ? 64 : d <= 128 ? 128 : 256;
    p.rows = tq * (heads / kv_heads);
    const int64_t groups = batch * kv_heads;
    if (p.rows > INT32_MAX / 8 || groups > INT32_MAX / 8) return -1;
    // Tiles of 32 rows fill the chip with fewer queries, tiles of 128 read keys a quarter as often. BF16, heads of 128: 3000 queries
    // of 8 heads on 4 (752 tiles of 32), a window of 127 behind them 18 against 11 us, of 1023 36 and 32; 2048 queries (512) 11 and
    // 11, 23 against 31; 4 clips of 750, 128 to both sides (768) 19 and 17, 2 (384) 12 against 16. FP32's matrix instructions take
    // longer than the reads: heads of 64, 1024 tiles 91 and 86 (1023 behind), heads of 128, 1500 tiles 281 against 337.
    const int64_t most_few = dtype != KEA_F32 ? 640 : p.dp > 64 ? 2560 : 1024;
    p.few = p.rows <= 64 || (p.rows + 31) / 32 * groups <= most_few;
    const int64_t per = p.few ? 32 : 128;
    p.row_tiles = (int)((p.rows + per - 1) / per);
    const int64_t wgs = p.row_tiles * groups;
    // the keys that a tile of rows can meet
    const int64_t most = 1 << 30, span = per / (heads / kv_heads) + 2;
    const int64_t window = left >= most || right >= most ? tk : left + right + span + (sinks < tk ? sinks : tk);
    const int64_t keys = window < tk ? window : tk;
    const int64_t tile = dtype == KEA_F32 ? (p.dp == 64 ? 128 : p.dp == 128 ? 64 : 32) : p.dp == 256 ? 64 : 128;
    const int64_t blocks = (keys + tile - 1) / tile;
    p.splits = 1;
    // Parts, where tiles of 32 rows leave CUs idle (one part more at 256 workgroups of four waves: BF16, heads of 128, 20 us
    // against 16), or SIMDs, where a workgroup has one or two waves and no form of four (heads of 129 to 256). FP32, heads of 65
    // to 128, has one from 129 workgroups on (750 frames of 8 heads, 128 to both sides, 26 us against 31 in two parts of two
    // waves). The second launch takes as long as two or three tiles of keys, and parts of 128 rows are long: BF16, 240 such
    // tiles 16 us whole, 27 in two parts.
    const int64_t most_split = p.dp == 256 ? 256 : p.dp == 128 && dtype == KEA_F32 ? 128 : 255;
    if (p.few && wgs > 0 && wgs <= most_split && blocks > 3) {
        int64_t s = 512 / wgs;  // up to two workgroups a CU
        s = s < blocks ? s : blocks;
        p.splits = (int)(s < 64 ? s : 64);
    }
    if (p.splits > 1) {
        p.part_bytes = p.splits * groups * p.rows * d * 4;
        p.stats_bytes = p.splits * groups * p.rows * 8;
    }
    *out = p;
    return 0;
}

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_window_attention: ") + hipGetErrorString(e));
}

template <typename T, int DP, int WQ, int WK, bool RAGGED>
int run_shape(const Args &a, hipStream_t stream) {
    using S = Shape<T, DP, WQ, WK>;
    static_assert(S::LDS <= 160 * 1024 && S::KT * S::UNITS % S::NT == 0 && S::KB <= 8, "tiles and flags");
    const int64_t groups = (int64_t)a.batch * a.kv_heads, padded = a.by_group ? (groups + 7) / 8 * 8 : a.row_tiles < 8 ? a.row_tiles : (a.row_tiles + 7) / 8 * 8;
    const dim3 grid((unsigned)padded, (unsigned)(a.by_group ? a.row_tiles : groups), (unsigned)a.splits);
    if (!kea::fits_dispatch(padded, S::NT) || grid.y > 65535 || !kea::fits_dispatch((int64_t)a.rows * (a.d / 4) / 64 + 1, 64))
        return kea::fail(KEA_EINVAL, "kea_window_attention: too large for one launch");
    const auto kernel = window_kernel<T, DP, WQ, WK, RAGGED>;
    const int lds = S::LDS;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return kea::fail((int)e, std::string("kea_window_attention: ") + hipGetErrorString(e));
    }
    kernel<<<grid, S::NT, lds, stream>>>(a);
    const int rc = launched();
    if (rc || a.splits == 1) return rc;
    join_kernel<T><<<dim3((unsigned)((a.rows * (a.d / 4) + 63) / 64), (unsigned)groups), 64, 0, stream>>>(a);
    return launched();
}

template <typename T, int DP>
int run_heads(const Args &a, bool few, hipStream_t stream) {
    if constexpr (sizeof(T) == 4 && DP == 128) {
        // Four waves in place of two, alone on their CU (128 KB of LDS), where all workgroups find one: 750 frames of 8 heads, 16 to
        // both sides, 14 against 20 us, 4 clips of 125 14 against 17; with 384 workgroups of five tiles 45 against 37.
        const int64_t wgs = (int64_t)a.row_tiles * a.batch * a.kv_heads;
        if (few && a.splits == 1 && wgs <= 256) return a.d == DP ? run_shape<T, DP, 1, 4, false>(a, stream) : run_shape<T, DP, 1, 4, true>(a, stream);
    }
    // waves that share out keys: four of them where two buffers of their blocks fit LDS
    constexpr int WK = 2 * 2 * 4 * 32 * DP * (int)sizeof(T) <= 131072 ? 4 : 2 * 2 * 2 * 32 * DP * (int)sizeof(T) <= 131072 ? 2 : 1;
    if (a.d == DP) return few ? run_shape<T, DP, 1, WK, false>(a, stream) : run_shape<T, DP, 4, 1, false>(a, stream);
    return few ? run_shape<T, DP, 1, WK, true>(a, stream) : run_shape<T, DP, 4, 1, true>(a, stream);
}

template <typename T>
int run_type(const Args &a, const Plan &p, hipStream_t stream) {
    return p.dp == 64 ? run_heads<T, 64>(a, p.few, stream) : p.dp == 128 ? run_heads<T, 128>(a, p.few, stream)
                                                                                 : run_heads<T, 256>(a, p.few, stream);
}

bool heads_ok(const kea_heads *t, int64_t unit) {
    return t && t->batch_stride >= 0 && t->t_stride >= 0 && t->head_stride >= 0 && (uintptr_t)t->data_dev % 16 == 0 && t->batch_stride % unit == 0 && t->t_stride % unit == 0 && t->head_stride % unit == 0;
}

int check_sizes(const char *what, int dtype, int64_t batch, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d,
                int64_t left, int64_t right, int64_t sinks, Plan *p) {
    if (dtype != KEA_F32 && dtype != KEA_F16 && dtype != KEA_BF16) return kea::fail(KEA_EINVAL, std::string(what) + ": f32, f16 or bf16");
    if (batch < 0 || tq < 0 || tk < 0 || tq > (1 << 30) || tk > (1 << 30) || heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 65535 || batch > (1 << 30))
        return kea::fail(KEA_EINVAL, std::string(what) + ": batch >= 0, 0 <= tq, tk <= 2^30 and heads a multiple of kv_heads are needed");
    if (d < 8 || d > 256 || d % 8) return kea::fail(KEA_EINVAL, std::string(what) + ": d is a multiple of 8 from 8 to 256");
    if (left < 0 || right < 0 || sinks < 0) return kea::fail(KEA_EINVAL, std::string(what) + ": left, right and sinks are >= 0");
    if (plan_of(dtype, batch, tq, tk, heads, kv_heads, d, left, right, sinks, p)) return kea::fail(KEA_EINVAL, std::string(what) + ": too large for one launch");
    return KEA_OK;
}

}  // namespace

extern "C" {

int64_t kea_window_attention_workspace(int dtype, int64_t batch, int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d,
                                       int64_t left, int64_t right, int64_t sinks) {
    Plan p;
    const int rc = check_sizes("kea_window_attention_workspace", dtype, batch, tq, tk, heads, kv_heads, d, left, right, sinks, &p);
    return rc ? rc : p.part_bytes + p.stats_bytes;
}

int kea_window_attention(const kea_heads *q, const kea_heads *k, const kea_heads *v, const kea_heads *out, int dtype, int64_t batch,
                         int64_t tq, int64_t tk, int64_t heads, int64_t kv_heads, int64_t d, int64_t left, int64_t right,
                         int64_t sinks, float scale, const int32_t *kv_lengths, const int32_t *q_starts, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    Plan p;
    const int rc = check_sizes("kea_window_attention", dtype, batch, tq, tk, heads, kv_heads, d, left, right, sinks, &p);
    if (rc) return rc;
    const int64_t unit = dtype == KEA_F32 ? 4 : 8;
    if (!heads_ok(q, unit) || !heads_ok(k, unit) || !heads_ok(v, unit) || !heads_ok(out, unit) || (uintptr_t)kv_lengths % 4 || (uintptr_t)q_starts % 4)
        return kea::fail(KEA_EALIGN, "kea_window_attention: pointers and strides are multiples of 16 bytes, strides not negative");
    if (!std::isfinite(scale)) return kea::fail(KEA_EINVAL, "kea_window_attention: the scale is not finite");
    if (batch == 0 || tq == 0) return KEA_OK;
    if (!q->data_dev || !out->data_dev || (tk > 0 && (!k->data_dev || !v->data_dev))) return kea::fail(KEA_EINVAL, "kea_window_attention: a pointer is missing");
    if (workspace_bytes < p.part_bytes + p.stats_bytes || (p.splits > 1 && !workspace)) return kea::fail(KEA_ESPACE, "kea_window_attention: the workspace is too small");
    if ((uintptr_t)workspace % 16) return kea::fail(KEA_EALIGN, "kea_window_attention: the workspace is aligned to 16 bytes");
    const int64_t most = 1 << 30;
    auto divide = [](uint64_t by, uint32_t *mul, uint32_t *shift) {
        for (*shift = 0; (1ULL << *shift) < by;) ++*shift;
        *mul = (uint32_t)((1ULL << (31 + *shift)) / by + 1);
    };
    uint32_t group_mul, group_shift, heads_mul, heads_shift;
    divide((uint64_t)(heads / kv_heads), &group_mul, &group_shift);
    divide((uint64_t)kv_heads, &heads_mul, &heads_shift);
    const int by_group = batch * kv_heads >= 8 && p.row_tiles <= 65535;
    const Args a{*q, *k, *v, *out, kv_lengths, q_starts, (float *)workspace, workspace ? (float *)((char *)workspace + p.part_bytes) : nullptr,
                 (int)batch, (int)tq, (int)tk, (int)kv_heads, (int)(heads / kv_heads), (int)d, (int)(left < most ? left : most),
                 (int)(right < most ? right : most), (int)(sinks < most ? sinks : most), (int)p.rows, p.row_tiles, p.splits, by_group,
                 group_mul, group_shift, heads_mul, heads_shift, scale};
    const hipStream_t s = (hipStream_t)stream;
    return dtype == KEA_F32 ? run_type<float>(a, p, s) : dtype == KEA_F16 ? run_type<_Float16>(a, p, s) : run_type<__bf16>(a, p, s);
}

}  // extern "C"
