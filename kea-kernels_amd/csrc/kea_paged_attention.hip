// Attention of new tokens over an int8 cache in pages (include/kea_decode.h).
//
// The query heads that share a key head are rows of one problem: row r of a sequence and key head is its new token r / group, head
// r % group of the group. Keys are walked once, 32 at a time, in products of 16-bit floats on whole numbers:
//   S^T = K Q^T        keys are the matrix instruction's rows, queries its columns, keys and values their codes -127 .. 127, exact in
//                      FP16: a lane holds 16 keys' sums of one query (its column)
//   s = S^T a          a = scale log2(e) k_scale, a number for each key (but for powers of two)
//   w = 2^(s - ref) v_scale, rounded to FP16;   O^T += V^T w^T;   l += 2^(s - top);   out = O 2^(ref - top) / l
// The queries are FP16 numbers: F16 as they are, BF16 by a power of two of their row (an element below 2^-28 of the row's largest is
// rounded to a multiple of 2^-28 of it), F32 the same in two parts, 22 bits of each element. The weights of F32 are in two parts too.
// The reference ref is such that w is below 2^15.94: it is raised, and O rescaled, only where a block's largest s + (exponent of that
// key's v_scale) passes it by more than 5.94 (base 2), and then stands where the largest w is 2^6 at least. Weights below 2^-14 lose digits of
// FP16: they are 2^-20 and less of the largest. Where the exponents of a block's v_scales are at most 3 apart, the largest s and the
// largest exponent are taken for it, of whichever keys they are; where they lie further apart, a key of no weight with a large
// v_scale would push the others' weights out of FP16's range, and each key's own sum is formed.
// The sum l has a reference of its own, the largest s so far, passed by 5.94 at most. Both are whole numbers: 2^(ref - top) is exact. One
// exponential serves both, 2^(s - ref), its sum times 2^(ref - top), while that factor is from 2^-100 to 2^60; beyond (values above some
// 2^70 or below 2^-90, and scores above 2^20) it would pass FP32's range or digits, and each has its own.
//
// Keys that a query does not see have p = 0, whatever scales they have: a scale of a key that no query sees is taken as 0, one that is
// no number makes the scores of its key NaN, for the queries that see it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "kea_attend.h"
#include "kea_internal.h"
#include "kea_pages.h"
#include "../../include/kea_decode.h"

namespace {

using kea::both_halves;
using kea::lptr_t;
using kea::other_half_max;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v2i *ltr8_t;
typedef __attribute__((address_space(3))) v4s *ltr16_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 5.9375f;  // what a block may pass the reference by (base 2) before it is raised
constexpr int kTop = 10;        // the exponent of the largest weight where the reference has just been raised: 2^(kTop + kLazy) < 65504
constexpr int kWide = 3;        // exponents of a block's value scales that are further apart are taken key by key
constexpr int kLeast = -149;    // the exponent that a value scale of zero counts as: below that of all others
constexpr float kNone = -0x1.fffffep127f;       // no reference yet: the lowest number
constexpr float kLarge = 0x1p20f;               // the largest reference that whole numbers up to some 2^8 are added to
constexpr int kFar = 60, kNear = -100;  // the largest and smallest ref - top with which one exponential serves both

struct Args {
    kea_heads q, out;
    kea_pages kp, vp;
    kea::Paging at;
    float *part, *stats;  // splits > 1: [splits][tokens][heads][d], [splits][tokens][heads][2]
    int kv_heads, group, d, left, splits, tiles_each, tiles;  // tiles_each: of a sequence, without offsets; tiles: the most there can be
    int fill;  // rows of no sequence become zeros
    float scale;  // times 2^by of each score
    int by;
};

// ---- what both kernels do --------------------------------------------------------------------------------------------------------

// A tile: rows r0 .. r0 + count - 1 of sequence b, whose first new token is row `first` of q and stands at position `start`.
struct Tile {
    int b, r0, rows, first, start, len;
};

// Tile `at` of PER rows; false where there are no more, with t->b the number that there are (with offsets). All values are uniform.
template <int PER>
__device__ __forceinline__ bool find_tile(const Args &a, int at, Tile *t) {
    int tile;
    if (!a.at.offsets) {
        t->b = at / a.tiles_each;
        tile = at - t->b * a.tiles_each;
        if (t->b >= a.at.batch) return false;
    } else {
        const int lane = __lane_id();
        int before = 0, found = -1;
        for (int j = 0; j < a.at.batch; j += 64) {
            int2 r = make_int2(0, 0);
            if (j + lane < a.at.batch) r = a.at.rows(j + lane);
            const int own = ((r.y - r.x) * a.group + PER - 1) / PER;
            int sum = own;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const int other = __shfl_up(sum, o);
                sum += lane >= o ? other : 0;
            }
            const uint64_t past = __ballot(before + sum > at);
            if (past) {
                const int l = __builtin_ctzll(past);
                found = j + l;
                tile = at - (before + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(own, l));
                break;
            }
            before += __builtin_amdgcn_readlane(sum, 63);
        }
        t->b = found < 0 ? before : found;
        if (found < 0) return false;
    }
    t->b = __builtin_amdgcn_readfirstlane(t->b);
    const int2 r = a.at.rows(t->b);
    t->first = __builtin_amdgcn_readfirstlane(r.x);
    const int n = __builtin_amdgcn_readfirstlane(r.y - r.x);
    t->rows = n * a.group;
    // the last tiles of a sequence see the most keys: they come first
    tile = __builtin_amdgcn_readfirstlane(tile);
    t->r0 = ((t->rows + PER - 1) / PER - 1 - tile) * PER;
    t->len = __builtin_amdgcn_readfirstlane(a.at.length(t->b));
    t->start = t->len - n;
    return true;
}

// Zeros for the rows of no sequence, of the heads of one key head: what workgroup `part` of the `parts` that found no tile does of it
// (4096 padded rows of 16 heads of 128 beside 8 tokens of 4000 keys: 93 us in all, 1072 with one workgroup for each key head's).
template <typename T>
__device__ void fill_rest(const Args &a, int hk, int threads, int part, int parts) {
    const int from = min(max(a.at.offsets[0], 0), a.at.tokens), to = min(max(a.at.offsets[a.at.batch], from), a.at.tokens);
    constexpr int E = 16 / sizeof(T);
    const int units = a.d / E, per = a.group * units;  // (vectors of a head, of a row)
    const long long all = (long long)(a.at.tokens - (to - from)) * per;
    for (long long i = (long long)part * threads + threadIdx.x; i < all; i += (long long)parts * threads) {
        const int row = (int)(i / per), e = (int)(i - (long long)row * per), t = row < from ? row : row + (to - from);
        *(v4f *)((T *)a.out.data_dev + (long long)t * a.out.t_stride + (long long)(hk * a.group + e / units) * a.out.head_stride + e % units * E) = v4f{0, 0, 0, 0};
    }
}

// Eight codes as FP16 numbers: 0x6400 + u is 1024 + u, u = code + 128.
__device__ __forceinline__ v8h numbers(uint32_t a, uint32_t b) {
    a ^= 0x80808080u, b ^= 0x80808080u;
    v4u w;
    w[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    w[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    w[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    w[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    const _Float16 less = (_Float16)1152.0f;
    return __builtin_bit_cast(v8h, w) - v8h{less, less, less, less, less, less, less, less};
}

__device__ __forceinline__ v16f mma(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// The exponent e with 2^(e - 1) <= |v| < 2^e; 0 for 0, infinities and NaN.
__device__ __forceinline__ int exponent(float v) { return __builtin_amdgcn_frexp_expf(v); }
// That of a value scale, as the reference takes it.
__device__ __forceinline__ int scale_exponent(float v) { return v != 0.0f ? exponent(v) : kLeast; }
__device__ __forceinline__ bool finite(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) != 0x7F800000u; }

// The largest number of each 16 lanes, in all of them; of 32 lanes (both halves of the wave hold the same ones).
__device__ __forceinline__ int row_max(int v) {
    auto dpp = [](int v, auto ctrl) { return __builtin_amdgcn_update_dpp(v, v, decltype(ctrl)::value, 0xF, 0xF, false); };
    v = max(v, dpp(v, std::integral_constant<int, 0xB1>{}));
    v = max(v, dpp(v, std::integral_constant<int, 0x4E>{}));
    v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));
    return max(v, dpp(v, std::integral_constant<int, 0x140>{}));
}
__device__ __forceinline__ int max32(int v) {
    v = row_max(v);
    return max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}

// A row of queries as the product's second operand, eight elements at a time; `at(i)` is the first element of operand i of this
// lane. *by: what a sum with it is multiplied by, a power of two: that of the row, and 2^up. (Rows whose power would not be a
// normal number with that are scaled by less: none of it is lost.)
template <typename T, int N, typename At>
__device__ __forceinline__ void load_queries(const T *row, int d, bool inside, At at, int up, v8h (&q)[N * (sizeof(T) == 4 ? 2 : 1)], float *by) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    auto load = [&](int i, float *v) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
        for (int u = 0; u < 8 / E; ++u) {
            const vec x = *(const vec *)(row + at(i) + u * E);
#pragma unroll
            for (int e = 0; e < E; ++e) v[u * E + e] = (float)x[e];
        }
    };
    int less = 0;
    if constexpr (!__is_same(T, _Float16)) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!inside || at(i) >= d) continue;
            float v[8];
            load(i, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, finite(v[e]) ? fabsf(v[e]) : 0.0f);
        }
        less = min(max(exponent(other_half_max(most)) - 5, -126 - up), 127 - up);
    }
    *by = __builtin_amdgcn_ldexpf(1.0f, less + up);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (!inside || at(i) >= d) {
#pragma unroll
            for (int p = 0; p < PARTS; ++p) q[i * PARTS + p] = v8h{0, 0, 0, 0, 0, 0, 0, 0};
            continue;
        }
        if constexpr (__is_same(T, _Float16)) {
            q[i] = *(const v8h *)(row + at(i));
        } else {
            float v[8];
            load(i, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = __builtin_amdgcn_ldexpf(v[e], -less);
                q[i * PARTS][e] = (_Float16)x;
                if constexpr (PARTS == 2) q[i * PARTS + 1][e] = (_Float16)(finite(x) ? x - (float)q[i * PARTS][e] : 0.0f);
            }
        }
    }
}

// a - b of two references, whole numbers; so far down where they are far apart that nothing is left of a product with its power.
__device__ __forceinline__ int difference(float a, float b) { return (int)fmaxf(a - b, -1000.0f); }

// The running references of a lane's query, its sum (of this half's keys) and what a block's sum of 2^(s - ref) takes part in it by.
struct Sums {
    float top = kNone, ref = kNone, l = 0.0f, unit = 1.0f;
    int up = 0;        // ref is top + up (to FP32: where that is not exact, the query is far)
    bool far = false;  // up is beyond kNear .. kFar, or top beyond kLarge: the sum and the weights have an exponential each
};

// What the sums make of a product: out = O 2^(ref - top) / l.
__device__ __forceinline__ v4f mean(v4f o, const Sums &m) {
    const float inv = m.l != 0.0f ? 1.0f / m.l : 0.0f;
    v4f v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(o[e] * inv, m.up);
    return v;
}
// Of several means: mean[s] 2^(top[s] - top) by (l[s] / the sum of l 2^(top[s] - top)), `by` the latter. (In this order neither a large value
// of next to no weight is lost nor anything passes FP32's range.)
__device__ __forceinline__ v4f portion(v4f mean, int down, float by) {
    v4f v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(mean[e], down) * by;
    return v;
}

// A block that some of a wave's rows do not see as a whole: what this lane's query does not see becomes -infinity. valid: the block's
// keys that have a page; hi, lo: the last and first key that the query sees, counted from the block's first. *v_exponent, *wide: as
// weigh takes them, of what this query sees.
__device__ __forceinline__ void mask(v16f &s, const v4f *v, uint32_t valid, int hi, int lo, int h, int *v_exponent, bool *wide) {
    asm volatile("");  // (a branch: not done for every block)
    const int hx = hi - 4 * h, lx = lo - 4 * h;
    const uint32_t bits = valid >> (4 * h);
    float most = 0.0f, less = -INFINITY;  // (the smallest as a largest: of the numbers below zero)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int at = 8 * (e / 4) + e % 4;
        const bool seen = at <= hx && at >= lx && (bits >> at & 1);
        if (!seen) s[e] = -INFINITY;
        most = fmaxf(most, seen ? fabsf(v[e / 4][e % 4]) : 0.0f);
        less = fmaxf(less, seen ? -fabsf(v[e / 4][e % 4]) : -INFINITY);
    }
    most = other_half_max(most), less = other_half_max(less);
    *v_exponent = scale_exponent(most);
    *wide = less != -INFINITY && scale_exponent(less) < *v_exponent - kWide;
}

// A block's scores s (16 keys of one query) become weights: in the sum, and times v as operands of the second product. v: the keys'
// value scales, v_exponent: the exponent of the largest of them, wide: some are more than kWide below it; by: what the scores are
// multiplied by. (s and v may be changed.)
template <int PARTS, int DB>
__device__ __forceinline__ void weigh(v16f &s, v4f *v, float by, int v_exponent, bool wide, Sums *m, v16f (&o)[DB], v4u (&w)[2 * PARTS]) {
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
    top = other_half_max(top) * by;
    const float less = (float)(v_exponent - kTop);
    bool passed = top + less > m->ref + kLazy || top > m->top + kLazy;
    float ref = m->ref;
    // (what few blocks need lies behind the loop: in line it took 10 % more for many rows)
    if (__builtin_expect(__any(passed || wide || m->far), 0)) {
        passed = passed || wide || m->far;
        const float next = passed ? floorf(fmaxf(m->top, top)) : m->top;
        const int down = difference(m->top, next);
        float own = top - next + (float)v_exponent;
        if (__any(wide)) {  // the largest over each key's own score and exponent
            float most = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) most = fmaxf(most, __builtin_fmaf(s[e], by, -next) + (float)scale_exponent(v[e / 4][e % 4]));
            most = other_half_max(most);
            own = wide ? most : own;
        }
        const int up = passed ? max(m->up + down, (int)fmaxf(floorf(own), -1000.0f) - kTop) : m->up;
        if (__any(m->top != kNone)) {  // (nothing is there to rescale at first)
            const float all = __builtin_amdgcn_ldexpf(1.0f, m->up + down - up);
            m->l = __builtin_amdgcn_ldexpf(m->l, down);
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= all;
        }
        m->top = next, m->up = up, m->ref = ref = next + (float)up;
        m->far = up > kFar || up < kNear || (fabsf(next) > kLarge && next != kNone);
        m->unit = m->far ? 0.0f : __builtin_amdgcn_ldexpf(1.0f, up);
    }
    if (__builtin_expect(__any(m->far), 0)) {  // their weights take the values' mantissas, with the values' exponents in the exponential
        float apart = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float x = v[e / 4][e % 4], t = __builtin_fmaf(s[e], by, -m->top);
            const int of_x = scale_exponent(x);
            apart += __builtin_amdgcn_exp2f(t);
            s[e] = m->far ? t + (float)(of_x - m->up) : s[e];
            v[e / 4][e % 4] = m->far ? __builtin_amdgcn_ldexpf(x, -of_x) : x;
        }
        by = m->far ? 1.0f : by, ref = m->far ? 0.0f : ref;
        m->l += m->far ? apart : 0.0f;
    }
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], by, -ref)), p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], by, -ref));
        float x0 = p0 * v[e / 4][e % 4], x1 = p1 * v[e / 4][e % 4 + 1];
        // (of two parts both are made from the FP32 product: the compiler may round the exact one to FP16 for the first)
        if constexpr (PARTS == 2) asm("" : "+v"(x0), "+v"(x1));
        sum += p0;
        sum += p1;
        const v2h hi = {(_Float16)x0, (_Float16)x1};
        w[e / 8 * PARTS][e % 8 / 2] = __builtin_bit_cast(uint32_t, hi);
        if constexpr (PARTS == 2) w[e / 8 * PARTS + 1][e % 8 / 2] = __builtin_bit_cast(uint32_t, v2h{(_Float16)(x0 - (float)hi[0]), (_Float16)(x1 - (float)hi[1])});
    }
    m->l = __builtin_fmaf(sum, m->unit, m->l);
}

template <typename T>
__device__ __forceinline__ void store4(T *y, v4f v) {
    T t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = (T)v[e];
    if constexpr (sizeof(T) == 4) *(v4f *)y = *(const v4f *)t;
    else *(v2u *)y = *(const v2u *)t;
}

// ---- few rows --------------------------------------------------------------------------------------------------------------------

// A workgroup takes up to 32 rows; its four waves take every fourth block of 32 keys each, on their own: a wave copies its blocks'
// codes and scales straight to LDS, NS - 1 blocks ahead, and no wave waits for another before the end, where their parts meet.
//
// A slot holds a block's keys, values (rows of DP bytes) and 32 scales of either. Unit u of 16 bytes of a row lies at u ^ f(key), so
// that neither the eight keys at one unit that eight lanes read as scores' operands, nor the eight keys at one unit that a
// transposing read takes, share banks.
//
// One token is bound by memory: 16 streams of up to 16000 BF16 keys of 4 heads of 128 are 176 MB of codes and scales, read in 50 us
// with the join as a graph of calls, 53 from call to call (3.5 and 3.3 TB/s; a large copy takes 33). For that 2 x 4 waves a CU have two
// blocks each under way; three or four blocks a wave leave room for one workgroup and take a third more (66 where two took 50). Without a barrier between them the waves drift apart, so that some load while others
// multiply.
template <int UNITS>
__device__ __forceinline__ int place(int key) {
    return UNITS == 4 ? (key >> 1 & 1) | ((key >> 2 ^ key >> 3) & 1) << 1 : (key & 7) ^ (key >> 3 & 1) << 2;
}

template <int DP, int NS>
struct Ring {
    static constexpr int UNITS = DP / 16, COPIES = UNITS / 2, KEYS = 32 * DP, SLOT = 2 * KEYS + 256, WAVE = NS * SLOT;
    static constexpr int MERGE = 4 * 32 * (DP + 2) * 4;
    static constexpr int LDS = 4 * WAVE > MERGE ? 4 * WAVE : MERGE;
};

template <typename T, int DP, int NS>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) token_kernel(Args a) {
    using R = Ring<DP, NS>;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, UNITS = R::UNITS, COPIES = R::COPIES, DB = DP / 32, QN = DP / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads, split = blockIdx.y;
    Tile t;
    if (!find_tile<32>(a, blockIdx.x / a.kv_heads, &t)) {
        if (a.fill && split == 0) fill_rest<T>(a, hk, 256, blockIdx.x / a.kv_heads - t.b, a.tiles + 1 - t.b);
        return;
    }
    const int count = min(32, t.rows - t.r0), row = min(t.r0 + n, t.rows - 1), token = row / a.group, head = hk * a.group + row - token * a.group;
    const int p = t.start + token, p0 = t.start + t.r0 / a.group, p1 = t.start + (t.r0 + count - 1) / a.group;
    const int hi = p, lo = max(0, p - a.left);

    // the blocks of 32 keys that some row sees, this split's and this wave's share of them
    const int first_key = max(0, p0 - a.left), block0 = first_key / 32, blocks = p1 < 0 ? 0 : p1 / 32 + 1 - block0;
    const int share = ((blocks + a.splits - 1) / a.splits + 3) / 4 * 4;
    const int from = min(blocks, split * share), to = min(blocks, from + share);
    const int steps = from + wave < to ? (to - from - wave + 3) / 4 : 0;
    if (to <= from && a.splits > 1) {  // nothing for this split
        if (tid < count) {
            const long long slot = ((long long)split * a.at.tokens + t.first + (t.r0 + tid) / a.group) * (a.kv_heads * a.group) + hk * a.group + (t.r0 + tid) % a.group;
            *(float2 *)(a.stats + 2 * slot) = make_float2(-INFINITY, 0.0f);
        }
        return;
    }

    // a lane's row and unit in the rows of one copy; the places of the units repeat every 16 keys
    constexpr int ROWS = 64 / UNITS, VARIANTS = 16 / ROWS;
    const uint32_t ring = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)lds + wave * R::WAVE);
    char *const own = lds + wave * R::WAVE;
    uint32_t off_k[VARIANTS], off_v[VARIANTS];
    bool some[VARIANTS];
#pragma unroll
    for (int u = 0; u < VARIANTS; ++u) {
        const int in = lane / UNITS, unit = (lane % UNITS) ^ place<UNITS>(u * ROWS + in);
        off_k[u] = (uint32_t)in * (uint32_t)a.kp.row_stride + 16 * unit;
        off_v[u] = (uint32_t)in * (uint32_t)a.vp.row_stride + 16 * unit;
        some[u] = 16 * unit < a.d;
    }
    const int8_t *const kd = a.kp.data_dev + (long long)hk * a.kp.head_stride, *const vd = a.vp.data_dev + (long long)hk * a.vp.head_stride;
    const float *const ks = a.kp.scale_dev + (long long)hk * a.kp.scale_head_stride, *const vs = a.vp.scale_dev + (long long)hk * a.vp.scale_head_stride;
    const int32_t *const table = a.at.table + (long long)t.b * a.at.table_stride;
    const int last_entry = a.at.width - 1, page_mask = (1 << a.at.shift) - 1;
    // the pages of the two halves of a block (uniform: read through the scalar cache)
    auto entries = [&](int step) {
        const int k0 = 32 * (block0 + from + wave + 4 * step);
        typedef const __attribute__((address_space(4))) int32_t *uniform_t;
        const uniform_t u = (uniform_t)(uintptr_t)table;
        return make_int2(u[min(k0 >> a.at.shift, last_entry)], u[min((k0 + 16) >> a.at.shift, last_entry)]);
    };
    auto stage = [&](int step, int2 page) {
        const int k0 = 32 * (block0 + from + wave + 4 * step);
        const uint32_t dst = ring + step % NS * R::SLOT;
        // (a half without a page is read from page 0, and masked)
        const int2 at = make_int2((unsigned)page.x < (unsigned)a.at.pages ? page.x : 0, (unsigned)page.y < (unsigned)a.at.pages ? page.y : 0);
        const int r0 = k0 & page_mask, r1 = (k0 + 16) & page_mask;
        const int8_t *const k_half[2] = {kd + at.x * a.kp.page_stride + r0 * a.kp.row_stride, kd + at.y * a.kp.page_stride + r1 * a.kp.row_stride};
        const int8_t *const v_half[2] = {vd + at.x * a.vp.page_stride + r0 * a.vp.row_stride, vd + at.y * a.vp.page_stride + r1 * a.vp.row_stride};
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
            const int key = c * ROWS;
            if (!some[c % VARIANTS]) continue;  // (units behind the row's end)
            kea::copy16(k_half[key / 16] + (key & 15) * a.kp.row_stride, off_k[c % VARIANTS], dst + c * 1024);
            kea::copy16(v_half[key / 16] + (key & 15) * a.vp.row_stride, off_v[c % VARIANTS], dst + R::KEYS + c * 1024);
        }
        const bool upper = n >= 16;
        const long long in_page = n & 15;
        const float *const k_from = ks + (upper ? at.y : at.x) * a.kp.scale_page_stride + ((upper ? r1 : r0) + in_page) * a.kp.scale_row_stride;
        const float *const v_from = vs + (upper ? at.y : at.x) * a.vp.scale_page_stride + ((upper ? r1 : r0) + in_page) * a.vp.scale_row_stride;
        kea::copy4(h ? v_from : k_from, dst + 2 * R::KEYS);
    };
    constexpr int COUNT = 2 * COPIES + 1;  // copies of a block
    static_assert(COUNT * (NS - 1) < 64, "vmcnt");
    auto landed = [&](int behind) {  // all copies but those of the last `behind` blocks
        asm volatile("" ::: "memory");
        auto wait = [&](auto left) {
            constexpr int LEFT = decltype(left)::value * COUNT;
            __builtin_amdgcn_s_waitcnt((LEFT & 15) | ((LEFT >> 4) << 14) | (15 << 8) | (7 << 4));
        };
        if (NS > 3 && behind >= 3) wait(std::integral_constant<int, (NS > 3 ? 3 : 0)>{});
        else if (NS > 2 && behind == 2) wait(std::integral_constant<int, (NS > 2 ? 2 : 0)>{});
        else if (behind == 1) wait(std::integral_constant<int, 1>{});
        else wait(std::integral_constant<int, 0>{});
        asm volatile("" ::: "memory");
    };

    int2 page[NS];  // of the blocks on their way, the next one to be computed first
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        page[s] = make_int2(-1, -1);
        if (s < NS - 1 && s < steps) {
            page[s] = entries(s);
            stage(s, page[s]);
        }
    }
    int2 next_page = NS - 1 < steps ? entries(NS - 1) : make_int2(-1, -1);

    v8h q[QN * PARTS];
    float by;
    load_queries<T, QN>((const T *)a.q.data_dev + (long long)(t.first + token) * a.q.t_stride + (long long)head * a.q.head_stride, a.d, p >= 0,
                        [&](int i) { return 16 * (2 * (i / 2) + h) + 8 * (i % 2); }, a.by, q, &by);

    v16f o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    Sums m;
    // operand addresses: unit 2 c + h of key n at ka ^ 32 c; eight keys' values of unit 2 d + (lane / 16) % 2, for the lanes' d
    const int ka = n * DP + (h ^ place<UNITS>(n)) * 16;
    const int vr = (lane & 15) >> 1, vkey = vr % 4 + 8 * (vr / 4) + 4 * h;
    const int va = vkey * DP + ((lane >> 4 & 1) ^ place<UNITS>(vkey)) * 16 + (lane & 1) * 8;

    for (int i = 0; i < steps; ++i) {
        // the block that follows those on their way, into the slot that has been read
        if (i + NS - 1 < steps) {
            page[NS - 1] = next_page;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            stage(i + NS - 1, next_page);
            if (i + NS < steps) next_page = entries(i + NS);
        }
        landed(min(NS - 1, steps - 1 - i));
        const int k0 = 32 * (block0 + from + wave + 4 * i);
        char *const slot = own + i % NS * R::SLOT;
        float *const scales = (float *)(slot + 2 * R::KEYS);

        // the scales: of keys that some row may see and that have a page, others 0; both rows are rewritten in place
        const uint32_t paged = ((unsigned)page[0].x < (unsigned)a.at.pages ? 0xFFFFu : 0u) | ((unsigned)page[0].y < (unsigned)a.at.pages ? 0xFFFF0000u : 0u);
        const int ahead = p1 - k0, behind = first_key - k0;  // the last and first key seen, in the block
        const uint32_t valid = paged & (ahead >= 31 ? ~0u : (2u << ahead) - 1u) & (behind > 0 ? ~0u << behind : ~0u);
        const float k_scale = scales[n], v_scale = scales[32 + n];
        const bool there = valid >> n & 1, number = finite(v_scale);
        const float x = !there ? 0.0f : number ? k_scale * a.scale * kLog2e : __builtin_nanf(""), y = there && number ? v_scale : 0.0f;
        const int own_exponent = scale_exponent(y);
        int v_exponent = max32(own_exponent);
        bool wide = __any(own_exponent < v_exponent - kWide);
        asm volatile("" ::: "memory");
        scales[lane] = h ? y : x;

        v16f s = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < QN / 2; ++c) {
            const v4u codes = *(const v4u *)(slot + (ka ^ 32 * c));
            const v8h k_lo = numbers(codes[0], codes[1]), k_hi = numbers(codes[2], codes[3]);
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                s = mma(k_lo, q[2 * c * PARTS + u], s);
                s = mma(k_hi, q[(2 * c + 1) * PARTS + u], s);
            }
        }
        asm volatile("" ::: "memory");
        v4f kx[4], vx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) kx[e] = *(const v4f *)(scales + 8 * e + 4 * h), vx[e] = *(const v4f *)(scales + 32 + 8 * e + 4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= kx[e / 4][e % 4];
        if (!(valid == 0xFFFFFFFFu && k0 + 31 <= p0 && k0 >= p1 - a.left)) mask(s, vx, valid, hi - k0, lo - k0, h, &v_exponent, &wide);  // not seen as a whole by every row
        v4u w[2 * PARTS];
        weigh<PARTS, DB>(s, vx, by, v_exponent, wide, &m, o, w);
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const v2i codes = __builtin_amdgcn_ds_read_tr8_b64_v2i32((ltr8_t)(slot + R::KEYS + (va ^ 32 * d) + 16 * z * DP));
                const v8h v = numbers((uint32_t)codes[0], (uint32_t)codes[1]);
#pragma unroll
                for (int u = 0; u < PARTS; ++u) o[d] = mma(v, __builtin_bit_cast(v8h, w[z * PARTS + u]), o[d]);
            }
#pragma unroll
        for (int s1 = 0; s1 + 1 < NS; ++s1) page[s1] = page[s1 + 1];
    }
    m.l = both_halves(m.l);

    // the waves' means, their sums and those's references meet in LDS: [wave][32][DP], then [wave][32][2]
    float *const po = (float *)lds, *const ps = po + 4 * 32 * DP;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
    if (n < count) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int c = 8 * d + e / 2 + h;  // (units of four elements, moved by the row: 32 rows are written at once)
                *(v4f *)(po + ((wave * 32 + n) * (DP / 4) + (c ^ (n & 7))) * 4) = mean(v4f{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]}, m);
            }
        if (h == 0) *(float2 *)(ps + 2 * (wave * 32 + n)) = make_float2(m.top, m.l);
    }
    __syncthreads();
    for (int at = tid; at < count * (DP / 4); at += 256) {
        const int r = at / (DP / 4), c = at % (DP / 4);
        if (4 * c >= a.d) continue;
        float2 st[4];
        float top = -INFINITY, all = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) st[w] = *(const float2 *)(ps + 2 * (w * 32 + r)), top = fmaxf(top, st[w].x);
        v4f v = {0, 0, 0, 0};
        int down[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            down[w] = difference(st[w].x, top);
            all += __builtin_amdgcn_ldexpf(st[w].y, down[w]);  // (a NaN stays one)
        }
        const float inv = all != 0.0f ? 1.0f / all : 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) v += portion(*(const v4f *)(po + ((w * 32 + r) * (DP / 4) + (c ^ (r & 7))) * 4), down[w], st[w].y * inv);
        const int tt = (t.r0 + r) / a.group, hh = hk * a.group + (t.r0 + r) - tt * a.group;
        if (a.splits > 1) {
            const long long slot = ((long long)split * a.at.tokens + t.first + tt) * (a.kv_heads * a.group) + hh;
            *(v4f *)(a.part + slot * a.d + 4 * c) = v;
            if (c == 0) *(float2 *)(a.stats + 2 * slot) = make_float2(top, all);
        } else {
            store4((T *)a.out.data_dev + (long long)(t.first + tt) * a.out.t_stride + (long long)hh * a.out.head_stride + 4 * c, v);
        }
    }
}

// ---- many rows -------------------------------------------------------------------------------------------------------------------

// A workgroup takes 256 rows (128 of heads up to 64), 32 a wave, which share tiles of 64 keys: each thread loads codes of the next tile
// into registers while the present one is worked on, and writes them to the other of two buffers as FP16 numbers, so that they are
// unpacked once for all rows. Wave 0 does the same with the scales.
//
// The place of unit c (eight numbers) of a key's row is c ^ place: rows that are read together lie in different banks. Keys: eight
// (16) rows at one unit. Values: four rows at two neighbouring pairs of units, which stay pairs.
//
// Instruction issue bounds it: for 32 x 32 scores 16 matrix instructions and some 200 vector ones (the scale, the mask's test, the
// largest, exponential, sum, v_scale and conversion of 16 scores a lane, and unpacking's share), of which little runs beside them. 2048
// tokens of 16000, 16 heads of 128 on 4: 344 us, 730 TFLOP/s where a large product of 16-bit floats makes 1220, at 1.8 to 1.9 GHz under
// this load. With 128 rows the unpacking has a second wave's share (11 % more).
template <int UNITS>
__device__ __forceinline__ int place_k(int key) {
    return UNITS == 8 ? key >> 1 & 7 : key & 15;
}
template <int UNITS>
__device__ __forceinline__ int place_v(int key) {
    return UNITS == 8 ? (key >> 1 & 1) * 4 : (key & 3) * 4;
}

template <int DP>
struct Tiles {
    static constexpr int WQ = DP == 128 ? 8 : 4, NT = 64 * WQ, ROWS = 32 * WQ, KB = 2, KT = 32 * KB, ROW = 2 * DP, UNITS = DP / 8;
    static constexpr int KEYS = KT * ROW, BUF = 2 * KEYS + 2 * KT * 4 + 16, LDS = 2 * BUF;  // keys, values, scales of both, 2 (exponent) + wide of blocks
    static constexpr int LOADS = KT * (DP / 16) / NT;  // of 16 codes, by each thread, of keys and of values
};

template <typename T, int DP>
__global__ void __launch_bounds__(Tiles<DP>::NT, 2) rows_kernel(Args a) {
    using S = Tiles<DP>;
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, KB = S::KB, KT = S::KT, ROW = S::ROW, UNITS = S::UNITS, LOADS = S::LOADS, DB = DP / 32, QN = DP / 16;
    constexpr int GRANULES = KT / 16, NT = S::NT, ROWS = S::ROWS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads, split = blockIdx.y;
    Tile t;
    if (!find_tile<ROWS>(a, blockIdx.x / a.kv_heads, &t)) {
        if (a.fill && split == 0) fill_rest<T>(a, hk, NT, blockIdx.x / a.kv_heads - t.b, a.tiles + 1 - t.b);
        return;
    }
    const int count = min(ROWS, t.rows - t.r0), w0 = min(t.r0 + 32 * wave, t.rows - 1), w1 = min(t.r0 + 32 * wave + 31, t.rows - 1);
    const bool real = 32 * wave + n < count;
    const int row = min(t.r0 + 32 * wave + n, t.rows - 1), token = row / a.group, head = hk * a.group + row - token * a.group;
    const int p = t.start + token, hi = p, lo = max(0, p - a.left);
    const int p0 = t.start + w0 / a.group, p1 = t.start + w1 / a.group;  // of the wave's rows
    const int first_p = t.start + t.r0 / a.group, last_p = t.start + (t.r0 + count - 1) / a.group;
    const int wave_first = max(0, p0 - a.left);

    // the tiles of keys that some row sees, and this split's share of them
    const int first_key = max(0, first_p - a.left), start = first_key / KT, all = last_p < 0 ? 0 : last_p / KT + 1 - start;
    const int share = (all + a.splits - 1) / a.splits, from = start + min(all, split * share), to = start + min(all, (split + 1) * share);
    if (to <= from && a.splits > 1) {  // nothing for this split
        if (tid < count) {
            const long long slot = ((long long)split * a.at.tokens + t.first + (t.r0 + tid) / a.group) * (a.kv_heads * a.group) + hk * a.group + (t.r0 + tid) % a.group;
            *(float2 *)(a.stats + 2 * slot) = make_float2(-INFINITY, 0.0f);
        }
        return;
    }

    const int8_t *const kd = a.kp.data_dev + (long long)hk * a.kp.head_stride, *const vd = a.vp.data_dev + (long long)hk * a.vp.head_stride;
    const float *const ks = a.kp.scale_dev + (long long)hk * a.kp.scale_head_stride, *const vs = a.vp.scale_dev + (long long)hk * a.vp.scale_head_stride;
    const int32_t *const table = a.at.table + (long long)t.b * a.at.table_stride;
    const int last_entry = a.at.width - 1, page_mask = (1 << a.at.shift) - 1;
    // The pages of a tile's granules of 16 keys (uniform: read through the scalar cache).
    typedef int pages_t __attribute__((ext_vector_type(GRANULES)));
    auto entries = [&](int tile) {
        typedef const __attribute__((address_space(4))) int32_t *uniform_t;
        const uniform_t u = (uniform_t)(uintptr_t)table;
        pages_t e;
#pragma unroll
        for (int i = 0; i < GRANULES; ++i) e[i] = u[min((KT * tile + 16 * i) >> a.at.shift, last_entry)];
        return e;
    };
    auto page_ok = [&](int page) { return (unsigned)page < (unsigned)a.at.pages; };
    // this thread's codes: unit `unit` of the keys key0 + u STEP, which lie in one granule for a wave
    constexpr int PER = DP / 16, STEP = NT / PER;
    const int key0 = tid / PER, unit = tid % PER;
    const bool some = 16 * unit < a.d;
    v4u k_codes[LOADS], v_codes[LOADS];
    float k_scale = 0.0f, v_scale = 0.0f;
    auto load = [&](int tile, pages_t e) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int granule = __builtin_amdgcn_readfirstlane((u * STEP + key0) / 16);
            int page = e[0];
#pragma unroll
            for (int i = 1; i < GRANULES; ++i) page = granule == i ? e[i] : page;
            if (!page_ok(page)) page = 0;  // (read, and masked)
            const int r0 = (KT * tile + 16 * granule) & page_mask;
            const uint32_t in = (uint32_t)(u * STEP + key0) % 16;
            const int8_t *const k_from = kd + (page * a.kp.page_stride + r0 * a.kp.row_stride), *const v_from = vd + (page * a.vp.page_stride + r0 * a.vp.row_stride);
            k_codes[u] = v_codes[u] = v4u{0, 0, 0, 0};
            if (some) {
                k_codes[u] = *(const v4u *)(k_from + (in * (uint32_t)a.kp.row_stride + 16u * (uint32_t)unit));
                v_codes[u] = *(const v4u *)(v_from + (in * (uint32_t)a.vp.row_stride + 16u * (uint32_t)unit));
            }
        }
        if (wave == 0) {
            const int key = lane % KT, granule = key / 16;
            int page = e[0];
#pragma unroll
            for (int i = 1; i < GRANULES; ++i) page = granule == i ? e[i] : page;
            if (!page_ok(page)) page = 0;
            const long long r = (KT * tile + key) & page_mask;
            k_scale = ks[page * a.kp.scale_page_stride + r * a.kp.scale_row_stride];
            v_scale = vs[page * a.vp.scale_page_stride + r * a.vp.scale_row_stride];
        }
    };
    // the keys of a tile that have a page and that some row of the workgroup may see
    auto valid_keys = [&](int tile, pages_t e) {
        uint64_t valid = 0;
#pragma unroll
        for (int i = 0; i < GRANULES; ++i) valid |= page_ok(e[i]) ? 0xFFFFULL << (16 * i) : 0;
        const int ahead = last_p - KT * tile, behind = first_key - KT * tile;  // the last and first key seen, in the tile
        return valid & (ahead >= 63 ? ~0ULL : (2ULL << ahead) - 1) & (behind > 0 ? ~0ULL << behind : ~0ULL);
    };
    auto put = [&](int buf, uint64_t valid) {
        char *const to = lds + buf * S::BUF;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int key = u * STEP + key0;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                *(v8h *)(to + key * ROW + ((2 * unit + half) ^ place_k<UNITS>(key)) * 16) = numbers(k_codes[u][2 * half], k_codes[u][2 * half + 1]);
                *(v8h *)(to + S::KEYS + key * ROW + ((2 * unit + half) ^ place_v<UNITS>(key)) * 16) = numbers(v_codes[u][2 * half], v_codes[u][2 * half + 1]);
            }
        }
        if (wave == 0) {
            float *const scales = (float *)(to + 2 * S::KEYS);
            const int key = lane % KT;
            const bool there = valid >> key & 1, number = finite(v_scale);
            scales[key] = !there ? 0.0f : number ? k_scale * a.scale * kLog2e : __builtin_nanf("");
            const float y = there && number ? v_scale : 0.0f;
            scales[KT + key] = y;
            const int e = scale_exponent(y), most = row_max(e);  // of 16 keys
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int block = max(__builtin_amdgcn_readlane(most, 32 * kb), __builtin_amdgcn_readlane(most, 32 * kb + 16));
                const bool apart = (uint32_t)(__ballot(e < block - kWide) >> (32 * kb)) != 0;
                if (lane == 0) ((int *)scales)[2 * KT + kb] = 2 * block + apart;
            }
        }
    };

    v8h q[QN * PARTS];
    float by;
    load_queries<T, QN>((const T *)a.q.data_dev + (long long)(t.first + token) * a.q.t_stride + (long long)head * a.q.head_stride, a.d, p >= 0,
                        [&](int i) { return 16 * i + 8 * h; }, a.by, q, &by);
    v16f o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    Sums m;
    // operand addresses: unit 2 c + h of key n at ka ^ 32 c, units 4 d .. of the values' rows at va ^ 64 d
    const int ka = n * ROW + (h ^ place_k<UNITS>(n)) * 16;
    const int vkey = 4 * h + (lane & 15) / 4, va = vkey * ROW + ((2 * (lane >> 4 & 1) + (lane & 3) / 2) ^ place_v<UNITS>(vkey)) * 16 + (lane & 1) * 8;

    pages_t pages{};
    uint64_t valid = 0, next_valid = 0;
    if (from < to) {
        pages = entries(from);
        load(from, pages);
        valid = valid_keys(from, pages);
        put(0, valid);
        if (from + 1 < to) pages = entries(from + 1);
    }
    for (int tile = from; tile < to; ++tile) {
        __syncthreads();
        const int buf = (tile - from) & 1;
        if (tile + 1 < to) {
            load(tile + 1, pages);
            next_valid = valid_keys(tile + 1, pages);
            if (tile + 2 < to) pages = entries(tile + 2);
        }
        const char *const kt = lds + buf * S::BUF, *const vt = kt + S::KEYS;
        const float *const scales = (const float *)(vt + S::KEYS);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int k0 = KT * tile + 32 * kb;
            if (k0 > p1 || k0 + 31 < wave_first) continue;  // seen by none of the wave's rows
            v16f s = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < QN; ++c) {
                const v8h k = *(const v8h *)(kt + 32 * kb * ROW + (ka ^ 32 * c));
#pragma unroll
                for (int u = 0; u < PARTS; ++u) s = mma(k, q[c * PARTS + u], s);
            }
            v4f kx[4], vx[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) kx[e] = *(const v4f *)(scales + 32 * kb + 8 * e + 4 * h), vx[e] = *(const v4f *)(scales + KT + 32 * kb + 8 * e + 4 * h);
            const int block = __builtin_amdgcn_readfirstlane(((const int *)scales)[2 * KT + kb]);
            int v_exponent = block >> 1;
            bool wide = block & 1;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] *= kx[e / 4][e % 4];
            const uint32_t here = (uint32_t)(valid >> (32 * kb));
            if (!(here == 0xFFFFFFFFu && k0 + 31 <= p0 && k0 >= p1 - a.left)) mask(s, vx, here, hi - k0, lo - k0, h, &v_exponent, &wide);  // not seen as a whole by every row
            v4u w[2 * PARTS];
            weigh<PARTS, DB>(s, vx, by, v_exponent, wide, &m, o, w);
#pragma unroll
            for (int i = 0; i < 2 * DB; ++i) {
                const char *const at = vt + (va ^ 64 * (i % DB)) + (32 * kb + 16 * (i / DB)) * ROW;
                const v4s x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ltr16_t)at), x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ltr16_t)(at + 8 * ROW));
                const v8h v = __builtin_bit_cast(v8h, v8s{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]});
#pragma unroll
                for (int u = 0; u < PARTS; ++u) o[i % DB] = mma(v, __builtin_bit_cast(v8h, w[i / DB * PARTS + u]), o[i % DB]);
            }
        }
        if (tile + 1 < to) put(buf ^ 1, next_valid);
        valid = next_valid;
    }
    m.l = both_halves(m.l);
    if (!real) return;
    const long long slot = ((long long)split * a.at.tokens + t.first + token) * (a.kv_heads * a.group) + head;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int c = 32 * d + 2 * e + 4 * h;
            if (c >= a.d) continue;
            const v4f v = mean(v4f{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]}, m);
            if (a.splits > 1) *(v4f *)(a.part + slot * a.d + c) = v;
            else store4((T *)a.out.data_dev + (long long)(t.first + token) * a.out.t_stride + (long long)head * a.out.head_stride + c, v);
        }
    if (a.splits > 1 && h == 0) *(float2 *)(a.stats + 2 * slot) = make_float2(m.top, m.l);
}

// Joins the splits: out = sum_s f_s mean_s, f_s = l_s 2^(top_s - top) over their sum; four elements a thread, eight splits at a time.
template <typename T>
__global__ void __launch_bounds__(64) join_kernel(Args a) {
    const int heads = a.kv_heads * a.group, per = a.d / 4;
    const long long at = (long long)blockIdx.x * 64 + threadIdx.x, slot0 = at / per, all_rows = (long long)a.at.tokens * heads;
    if (slot0 >= all_rows) return;
    const int c = (int)(at - slot0 * per), t = (int)(slot0 / heads), head = (int)(slot0 - (long long)t * heads);
    if (a.at.offsets && !(t >= a.at.offsets[0] && t < a.at.offsets[a.at.batch])) return;
    float top = -INFINITY, all = 0.0f;
    v4f v = {0, 0, 0, 0};
    for (int s0 = 0; s0 < a.splits; s0 += 8) {
        float2 st[8];
        v4f part[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const long long slot = min(s0 + s, a.splits - 1) * all_rows + slot0;
            st[s] = *(const float2 *)(a.stats + 2 * slot);
            part[s] = *(const v4f *)(a.part + slot * a.d + 4 * c);
            if (s0 + s >= a.splits) st[s].y = 0.0f;
        }
        const float old = top;
#pragma unroll
        for (int s = 0; s < 8; ++s) top = fmaxf(top, st[s].x);
        float sum = __builtin_amdgcn_ldexpf(all, difference(old, top));
#pragma unroll
        for (int s = 0; s < 8; ++s) sum += __builtin_amdgcn_ldexpf(st[s].y, difference(st[s].x, top));
        // (the sum so far is kept as a mean: it neither overflows nor loses digits that the mean has)
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        v = portion(v, difference(old, top), all * inv);
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (st[s].y != 0.0f) v += portion(part[s], difference(st[s].x, top), st[s].y * inv);  // (a part that saw nothing was not written)
        all = sum;
    }
    store4((T *)a.out.data_dev + (long long)t * a.out.t_stride + (long long)head * a.out.head_stride + 4 * c, v);
}

// ---- host ----------------------------------------------------------------------------------------------------------------------

struct Plan {
    bool few;  // tiles of 32 rows
    int64_t tiles, tiles_each, splits, part_bytes, stats_bytes;
};

int plan_of(int64_t batch, int64_t tokens, int64_t positions, int64_t heads, int64_t kv_heads, int64_t d, int64_t left, bool offsets, Plan *out) {
    const int64_t group = heads / kv_heads, each = batch > 0 ? tokens / batch : 0;
    Plan p{};
    // The keys that a token may meet: the positions that there is room for (lengths are not known here), less what causality hides.
    const int64_t room = positions - each / 2, keys = left < room ? left + 1 : room;
    // Tiles of 32 rows walk their keys without a wait between waves, tiles of 256 unpack the codes for eight times as many rows: they
    // are ahead where there are many rows and long walks. F16, heads of 128, 16 on 4, us (32 rows, 256 rows): 2048 tokens of 16000
    // 502 and 346, 1000 of 16000 253 and 187, 8 x 512 of 4000 247 and 205, 1000 of 4000 67 and 66, 2048 of 4000 105 and 106, 4000 of
    // 4000 139 and 130, 2048 of 2048 47 and 68, 1000 of 1000 19 and 36; 512 of 4000 (FP32) 63 and 61. (A table with room for more keys
    // than its sequences hold counts as they would: a prompt of 2048 in a table of 16000 takes 256 rows.) Heads of 129 to 256 are faster
    // in 32 rows throughout (a tenth: the outputs of a row alone take half of a wave's registers).
    p.few = d > 128 || tokens * heads < 16000 || keys < 3000;
    const int64_t per = p.few ? 32 : d <= 64 ? Tiles<64>::ROWS : Tiles<128>::ROWS;
    p.tiles_each = (each * group + per - 1) / per;
    p.tiles = offsets ? tokens * group / per + batch : p.tiles_each * batch;
    if (tokens * group > INT32_MAX / 4 || p.tiles > INT32_MAX / 4) return -1;
    const int64_t wgs = p.tiles * kv_heads;
    p.splits = 1;
    if (wgs > 0 && p.few) {
        // Two workgroups on every CU where each part has 700 keys and more, one otherwise; 128 keys at least. BF16, one token of 16 streams
        // of 16000 keys (64 workgroups): 182, 102, 61, 56 and 59 us in 1, 2, 4, 8 and 16 parts; 64 tokens of 4000 (32) 52, 34, 25, 21 and 25;
        // 8 x 64 of 1000 (256) 22 and 30 in 1 and 2.
        const int64_t span = keys + per / group;
        int64_t s = wgs < 512 ? 512 / wgs : 1;
        if (span / s < 700) s = wgs < 256 ? 256 / wgs : 1;
        const int64_t most = (span + 127) / 128;
        s = s < most ? s : most;
        p.splits = s < 1 ? 1 : s < 64 ? s : 64;
    } else if (wgs > 0) {
        // One workgroup on every CU, or two rounds of them, whose parts even out what causality leaves to the tiles: 4000 of 4000 (256
        // workgroups) 170 us in one, 135 in two, 151 in four parts; 2048 of 16000 (128) 347 in two, 436 in three.
        const int64_t s = wgs <= 128 ? 256 / wgs : wgs < 384 ? 2 : 1;
        p.splits = s < 16 ? s : 16;
    }
    if (p.splits > 1) {
        p.part_bytes = p.splits * tokens * heads * d * 4;
        p.stats_bytes = p.splits * tokens * heads * 8;
    }
    *out = p;
    return 0;
}

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KEA_OK : kea::fail((int)e, std::string("kea_paged_attention: ") + hipGetErrorString(e));
}

// One of the two kernels, then the join of its parts.
int launch(void (*kernel)(Args), void (*join)(Args), int threads, int lds, const Args &a, hipStream_t stream) {
    const int64_t tiles = ((int64_t)a.tiles + a.fill) * a.kv_heads;
    const int64_t joins = ((int64_t)a.at.tokens * a.kv_heads * a.group * (a.d / 4) + 63) / 64;
    if (!kea::fits_dispatch(tiles, threads) || !kea::fits_dispatch(joins, 64)) return kea::fail(KEA_EINVAL, "kea_paged_attention: too large for one launch");
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return kea::fail((int)e, std::string("kea_paged_attention: ") + hipGetErrorString(e));
    }
    kernel<<<dim3((unsigned)tiles, (unsigned)a.splits), threads, lds, stream>>>(a);
    const int rc = launched();
    if (rc || a.splits == 1) return rc;
    join<<<dim3((unsigned)joins), 64, 0, stream>>>(a);
    return launched();
}

template <typename T, int DP, int NS>
int run_few(const Args &a, hipStream_t stream) {
    static_assert(Ring<DP, NS>::LDS <= 160 * 1024, "LDS");
    return launch(token_kernel<T, DP, NS>, join_kernel<T>, 256, Ring<DP, NS>::LDS, a, stream);
}

template <typename T, int DP>
int run_rows(const Args &a, hipStream_t stream) {
    using S = Tiles<DP>;
    static_assert(S::LDS <= 160 * 1024 && S::LOADS * S::NT == S::KT * (DP / 16) && S::LOADS > 0, "LDS and loads");
    return launch(rows_kernel<T, DP>, join_kernel<T>, S::NT, S::LDS, a, stream);
}

template <typename T>
int run(const Args &a, bool few, hipStream_t stream) {
    if (!few) return a.d <= 64 ? run_rows<T, 64>(a, stream) : run_rows<T, 128>(a, stream);
    return a.d <= 64 ? run_few<T, 64, 4>(a, stream) : a.d <= 128 ? run_few<T, 128, 2>(a, stream) : run_few<T, 256, 2>(a, stream);
}

bool rows_ok(const kea_heads *t, int64_t unit) {
    return t && t->t_stride >= 0 && t->head_stride >= 0 && (uintptr_t)t->data_dev % 16 == 0 && t->t_stride % unit == 0 && t->head_stride % unit == 0;
}

int check_sizes(const char *what, int dtype, int64_t batch, int64_t tokens, int64_t positions, int64_t heads, int64_t kv_heads, int64_t d,
                int64_t left, bool offsets, Plan *p) {
    const std::string name(what);
    if (dtype != KEA_F32 && dtype != KEA_F16 && dtype != KEA_BF16) return kea::fail(KEA_EINVAL, name + ": f32, f16 or bf16");
    if (batch < 0 || tokens < 0 || positions < 0 || batch >= (1 << 30) || tokens >= (1 << 30) || positions > (1 << 30) || heads < 1 || kv_heads < 1 || heads % kv_heads ||
        heads > 65535 || left < 0)
        return kea::fail(KEA_EINVAL, name + ": sizes are not negative and below 2^30, heads a multiple of kv_heads");
    if (d < 16 || d > 256 || d % 16) return kea::fail(KEA_EINVAL, name + ": d is a multiple of 16 from 16 to 256");
    if (plan_of(batch, tokens, positions, heads, kv_heads, d, left, offsets, p)) return kea::fail(KEA_EINVAL, name + ": too large for one launch");
    return KEA_OK;
}

}  // namespace

extern "C" {

int64_t kea_paged_attention_workspace(int dtype, int64_t batch, int64_t tokens, int64_t positions, int64_t heads, int64_t kv_heads, int64_t d,
                                      int64_t left, int offsets) {
    Plan p;
    const int rc = check_sizes("kea_paged_attention_workspace", dtype, batch, tokens, positions, heads, kv_heads, d, left, offsets != 0, &p);
    return rc ? rc : p.part_bytes + p.stats_bytes;
}

int kea_paged_attention(const kea_heads *q, const kea_heads *out, int dtype, int64_t heads, int64_t kv_heads, int64_t d, const kea_pages *k_pages,
                        const kea_pages *v_pages, const kea_paging *paging, int64_t left, float scale, int fill, void *workspace,
                        int64_t workspace_bytes, void *stream) {
    Args a{};
    const int bad = kea::check_paging("kea_paged_attention", k_pages, v_pages, paging, kv_heads, d, &a.at);
    if (bad) return bad;
    Plan p;
    const int rc = check_sizes("kea_paged_attention", dtype, paging->batch, paging->tokens, paging->table_width * paging->page_size, heads, kv_heads, d,
                               left, paging->q_offsets_dev != nullptr, &p);
    if (rc) return rc;
    const int64_t unit = dtype == KEA_F32 ? 4 : 8;
    if (!rows_ok(q, unit) || !rows_ok(out, unit)) return kea::fail(KEA_EALIGN, "kea_paged_attention: rows and their strides are multiples of 16 bytes, strides not negative");
    if (!std::isfinite(scale)) return kea::fail(KEA_EINVAL, "kea_paged_attention: the scale is not finite");
    if (k_pages->row_stride >= (1 << 26) || v_pages->row_stride >= (1 << 26)) return kea::fail(KEA_EINVAL, "kea_paged_attention: rows of a page 2^26 bytes and more apart");
    if (paging->tokens == 0) return KEA_OK;
    if (!q->data_dev || !out->data_dev) return kea::fail(KEA_EINVAL, "kea_paged_attention: a pointer is missing");
    if (workspace_bytes < p.part_bytes + p.stats_bytes || (p.splits > 1 && !workspace)) return kea::fail(KEA_ESPACE, "kea_paged_attention: the workspace is too small");
    if ((uintptr_t)workspace % 16) return kea::fail(KEA_EALIGN, "kea_paged_attention: the workspace is aligned to 16 bytes");
    a.q = *q, a.out = *out, a.kp = *k_pages, a.vp = *v_pages;
    a.part = (float *)workspace, a.stats = workspace ? (float *)((char *)workspace + p.part_bytes) : nullptr;
    a.kv_heads = (int)kv_heads, a.group = (int)(heads / kv_heads), a.d = (int)d, a.left = (int)(left < (1 << 30) ? left : 1 << 30);
    a.splits = (int)p.splits, a.tiles_each = (int)p.tiles_each, a.tiles = (int)p.tiles;
    // A score is (sum of codes and queries) (k_scale scale log2(e)) 2^by: the sum is below 2^20 (FP16 queries, which have no power of two
    // of their own, 2^31) and k_scale below 2^122, so that 2^-16 (2^-27) of the scale's power are left with them and the rest goes with the
    // queries'.
    int power = 0;
    std::frexp(scale, &power);
    a.by = std::min(std::max(power + (dtype == KEA_F16 ? 27 : 16), -126), 127);
    a.scale = std::ldexp(scale, -a.by);
    a.fill = fill && paging->q_offsets_dev ? 1 : 0;
    if (a.at.batch == 0 && !a.fill) return KEA_OK;  // (no tiles, and the rows of no sequence stay as they are)
    const hipStream_t s = (hipStream_t)stream;
    return dtype == KEA_F32 ? run<float>(a, p.few, s) : dtype == KEA_F16 ? run<_Float16>(a, p.few, s) : run<__bf16>(a, p.few, s);
}

}  // extern "C"
