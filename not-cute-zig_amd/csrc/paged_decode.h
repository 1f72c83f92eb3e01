// paged_decode.h — single-token attention over pages, shared by paged.hip (caches in 16 bits) and paged4.hip (in 4 bits, and
// those that add the weights up by token). What device memory names (lengths, page ids) is checked here before it becomes an
// address.
#ifndef NOTCUTE_PAGED_DECODE_H
#define NOTCUTE_PAGED_DECODE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "paged_args.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ uint32_t wave_scan32(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
    return x;
}
// Of numbers below 2^32, whose sums may pass that: their halves' sums do not.
__device__ __forceinline__ uint64_t wave_scan64(uint32_t x) {
    return wave_scan32(x & 0xffffu) + ((uint64_t)wave_scan32(x >> 16) << 16);
}

// Largest j in [0, n) with s[j] <= x, for s ascending and s[0] <= x; n is a power of two.
__device__ __forceinline__ uint32_t last_not_above(const uint32_t *s, uint32_t n, uint32_t x) {
    uint32_t j = 0;
    for (uint32_t step = n >> 1; step; step >>= 1)
        if (s[j + step] <= x) j += step;
    return j;
}

}  // namespace

// -------------------------------------------------------------------------------------------------
// Single-token attention. Up to 16 query heads of one key head are the 16 columns of the matrix products, so
// K and V are read once for all of them; with up to 64, two or four waves of a workgroup take the same keys at
// the same time, and all but one find them in the caches. The work is cut into blocks, counted over all requests
// and heads, and every workgroup takes a run of equally many, whatever the lengths: it finds its first by a
// prefix sum over the requests' lengths. A run that begins or ends inside a request's keys leaves a piece
// (max, sum, O), and the workgroups that arrive last add the pieces up, in rounds and in a fixed order. Heads of
// at most two blocks are not split, and where there are more heads than workgroups a wave takes a short one for itself.
// Where the heads of a token are next to each other (_next) and a request is long, two or four waves take neighbouring heads
// of the same keys, so that what shares a line or a row of memory is read at one time; their query heads are one piece.
//
// One wave takes KT x 32 keys of a block at a time. Scores: S = K Q^T with K rows straight from memory as the
// A operand (lane l: key l%16, dims 8(l/16)..+7 of 32), so lane l holds the scores of query l%16 and keys
// 4(l/16)+r of each 16. These registers are the B operand of O^T += V^T P^T as they stand, if V's k index runs
// the same way: the lane loads D/16 dims of the eight keys 16t + 4(l/16) + r and turns them in registers.
// Nothing but the final join of the four waves goes through LDS. K and V are read once and the rest is small, so
// the read rate bounds it; the matrix cores have time for weights in two (f16) or three (bf16) parts, whose
// sum is the f32 weight to 2^-21 or better (UNIT says down to which weight): rounding them to one 16-bit number would
// cost 2^-11 or 2^-8. The product with UNIT and the f16 parts' own accumulators cost 0 to 2 % (33 requests of up to 2047 over 16
// heads of 32 11.1 -> 11.4 us; 96 of 8192 over 8 of 128 537 on both sides).
//
// Measured in replayed graphs (bytes of K and V that count):
//   96 requests of 8192 over 8 heads of 128, 64 query heads    537 us  6.0 TB/s (a large copy moves 4.9)
//   one of 120001 over 8 heads of 64                            51     4.8      (token-major 54 to 56)
//   64 ragged ones of up to 16000 over 4 heads of 64            28.7   4.3
//   16 of 1000 over 8 of 128                                    16.4   4.0
//   one of 100                                                   4.4
// and in 4 bits (bytes of codes and scales; FOUR below):
//   96 requests of 8192 over 8 heads of 128, 64 query heads    165 us  5.2 TB/s (VALU 46 % busy)
//   one of 120001 over 8 heads of 64, token-major               32     2.0      (waits: 7 steps a wave)
//   16 of 1000 over 8 of 128                                    14.2   1.3
//   one of 100                                                   5.8
// Scores kept for the weights by token: 16 of 4096 over 8 of 128, 32 query heads, in 16 bits 59 us (53 without).
// The short ones are a chain of waits: launch, lengths, table, K and V, O, and for a piece the stores, the count and the
// others' pieces. More than 64 requests' lengths are read one after the other by a lane (4096 requests: 26 us).
// -------------------------------------------------------------------------------------------------
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
typedef short shortx2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx32 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// Memory that no kernel in flight writes, read by scalar loads.
typedef const __attribute__((address_space(4))) int32_t *const_ints;

__device__ __forceinline__ const_ints as_const(const int32_t *p) { return (const_ints)(uintptr_t)p; }

template <bool BF>
__device__ __forceinline__ floatx4 mfma_k32(u32x4 x, u32x4 y, floatx4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ floatx4 mfma_k16(u32x2 x, u32x2 y, floatx4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4v, x), __builtin_bit_cast(short4v, y), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4, x), __builtin_bit_cast(half4, y), c, 0, 0, 0);
}

// Two f32 rounded to nearest as a pair of 16-bit numbers; x and y become what that leaves, in f16 times kLowUnit: at most
// half a step of a number below 2^16, times 2^12 below 2^16 too, and exact.
constexpr float kLowUnit = 0x1p12f;
template <bool BF, bool ONCE = false>
__device__ __forceinline__ uint32_t take_pair(float &x, float &y) {
    if constexpr (BF) {
        const bf16x2 h = {(__bf16)x, (__bf16)y};
        uint32_t u = __builtin_bit_cast(uint32_t, h);
        if constexpr (ONCE) asm("" : "+v"(u));  // else it is converted again, by halves
        x -= __uint_as_float(u << 16);
        y -= __uint_as_float(u & 0xffff0000u);
        return u;
    } else {
        const half2v h = {(_Float16)x, (_Float16)y};
        x = (x - (float)h[0]) * kLowUnit;
        y = (y - (float)h[1]) * kLowUnit;
        return __builtin_bit_cast(uint32_t, h);
    }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false));
}
// Over each 4 neighbouring lanes, or each 16; all get the result.
template <bool MAX>
__device__ __forceinline__ float near(float x, bool sixteen) {
    auto add = [](float u, float v) { return MAX ? fmaxf(u, v) : u + v; };
    x = add(x, dpp<0xb1>(x));  // quad_perm 1,0,3,2 and 2,3,0,1
    x = add(x, dpp<0x4e>(x));
    if (sixteen) {
        x = add(x, dpp<0x124>(x));  // row_ror:4 and 8
        x = add(x, dpp<0x128>(x));
    }
    return x;
}

// Over the four lanes l, l^16, l^32, l^48; all get the result.
__device__ __forceinline__ float quad_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// Over the two lanes l, l^16.
__device__ __forceinline__ uint32_t pair_max(uint32_t x) {
    auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max((uint32_t)a[0], (uint32_t)a[1]);
}
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
    auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return pair_max(max((uint32_t)b[0], (uint32_t)b[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Partials go between workgroups of different XCDs, whose L2 caches are not coherent for ordinary accesses:
// relaxed atomics at agent scope are. Their order against the counter is made by waits (see join()).
__device__ __forceinline__ void put2(float *p, float x, float y) {
    const uint64_t v = (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void get2(const float *p, float &x, float &y) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = __uint_as_float((uint32_t)v);
    y = __uint_as_float((uint32_t)(v >> 32));
}

// The argument block where the launch put it. again() hides that it is the same one, so that what only a head's
// beginning or end needs is read there once more and does not stay in scalar registers: a few dozen too many of
// them were written to and read back from a vector register in every step.
typedef const __attribute__((address_space(4))) nc_paged_decode_args *Args;
__device__ __forceinline__ Args again(Args p) {
    asm volatile("" : "+s"(p));
    return p;
}

__device__ __forceinline__ float finite_or_0(float m) { return m == neg_inf() ? 0.f : m; }

// The arguments that kernels of 4-bit caches and those that keep scores have behind the common ones.
__device__ __forceinline__ const __attribute__((address_space(4))) nc_paged_more_args *more_of(Args a) {
    return reinterpret_cast<const __attribute__((address_space(4))) nc_paged_more_args *>(a);
}

// Two 4-bit values, byte b of w, times a power of two, as bf16: exact, and NaN where the scale's exponent field is 255.
__device__ __forceinline__ uint32_t pair_of_fours(uint32_t w, float scale, int b) {
    switch (b) {
        case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
        case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
        case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
        default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    }
}

// Parts of f32 values as small numbers times a power of two. x becomes what that leaves, exactly, which the next part takes with a scale 2^-5
// of this one (LAST: nothing asks for it). Four values of at most 2 scales as e4m3 bytes:
template <bool LAST>
__device__ __forceinline__ uint32_t take_eights(float (&x)[4], float scale) {
    shortx2 w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(shortx2{0, 0}, x[0], x[1], scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[2], x[3], scale, true);
    const uint32_t u = __builtin_bit_cast(uint32_t, w);
    if constexpr (!LAST) {
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(u, scale, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(u, scale, true);
        x[0] -= lo[0];
        x[1] -= lo[1];
        x[2] -= hi[0];
        x[3] -= hi[1];
    }
    return u;
}
// 32 values of at most 4 scales, x[i] and y[i] in turn, as e2m3 (eighths below 2, quarters below 4):
template <bool LAST>
__device__ __forceinline__ u32x6 take_sixes(floatx16 &x, floatx16 &y, float scale) {
    const u32x6 w = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(x, y, scale);
    if constexpr (!LAST) {
        const floatx32 z = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(w, scale);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] -= z[2 * i];
            y[i] -= z[2 * i + 1];
        }
    }
    return w;
}

// FOUR: the cache holds 4-bit values (e2m1) with a scale byte 2^(b - 127) for every 32 of a row. K rows are then the A operand
// of v_mfma_scale_f32_16x16x128_f8f6f4 as they lie in memory, codes and scales, and Q its B operand as the sum of
// small numbers, QPARTS each. Products are exact but for f32's rounding: the instruction adds those of 8
// neighbours in fixed point, which keeps 13 bits below the largest, all that products of e2m3 have, and of e4m3 of at most 2 (of up to 16
// the scores were off by 2^-13). V is
// turned into bf16, which holds every value of a 4-bit cache, and BF is true.
// MASS: every query head's scores are kept, and its maximum and sum, for the weights' kernel.
// PACK: where a key head has at most 8 or 4 query heads, the 16 columns are 2 or 4 groups of them, each with a maximum, a sum and an
// O of its own, that take every second or fourth tile: a step's scores then are half or a quarter of the registers.
template <int D, bool BF, bool UNI, bool MANY, bool NEXT, bool FOUR = false, bool MASS = false, int PACK = 1>
struct Decode {
    static_assert((BF && D >= 32) || !FOUR, "a 4-bit cache's V is bf16, and a group of 32 is a row's or part of it");
    static constexpr int KT = FOUR ? NC_PAGED4_STEP_KEYS / 32 : D <= 32 ? 2 : 1;  // 32-key tiles of a wave's step
    static constexpr int NT = 2 * KT;           // 16-key tiles
    // FOUR: parts of Q. Heads of 128 have 6-bit ones, whose products take half the time of 8-bit ones', and whose 32 dims that share a scale
    // are a lane's. With five of those and with four 8-bit ones: 96 requests of 8192 over 8 heads of 128 169.7 and 173.3 us, 16 of 1000
    // 14.0 and 14.4. Smaller heads' 8-bit products have columns to spare, and a lane half as much to split: one of 100 over 8 heads of 64 6.04 and
    // 5.77, 227 of up to 3464 over 8 of 32, whose split leaves room for fewer waves, 37.9 and 29.7.
    static constexpr bool SIXES = D == 128;
    static constexpr int QPARTS = SIXES ? 5 : 4;
    static constexpr int QDIMS = SIXES ? 32 : 16;  // dims of a lane
    static constexpr uint32_t WK = 32 * KT;     // keys of a wave's step
    static constexpr int E = D / 16;            // dims of a lane in V and O
    static constexpr int KK = FOUR ? QPARTS * D / 128 : D < 32 ? 1 : D / 32;  // products of a score
    static constexpr int KL = FOUR ? 1 : KK;    // loads of a row of K
    static constexpr uint32_t HEAD_UNITS = FOUR ? nc_paged4_head_units(D) : nc_paged_head_units(D);
    static constexpr int KE = D == 16 ? 4 : 8;  // dims of a lane in one product
    // Whether a step's loads are under way before the one before it is computed. It costs registers, and pays where a step's
    // loads are wide and heads end at different times: 64 ragged requests over 4 heads of 64 31.6 -> 28.7 us, 32 of 2048 over 8
    // of 64 28.0 -> 27.6 (but one of 120001 over 8 of 64, token-major, 53 -> 56). Heads of 16 or 32 are better off with more
    // workgroups instead (33 requests of up to 2047, 16 heads of 32, 11.9 -> 11.1 us on pages of 16, and 14.4 -> 11.4 of 7), and
    // with heads of 128 on odd pages both the addresses and two steps do not fit (1 % slower). 4-bit caches' steps are shorter and
    // two workgroups of a CU hide each other's (16 of 1000 over 8 heads of 128 16.6 -> 14.4 us without, 96 of 8192 191 -> 170).
    static constexpr bool AHEAD = !FOUR && (D == 64 || (D == 128 && UNI));
    static constexpr uint32_t COLS = 16 / PACK;  // query heads of a column group
    static constexpr int SETS = NT / PACK;       // tiles of a column group
    static constexpr int OP = D + 4;            // pitch of a row of partial O in LDS
    static constexpr uint32_t NW = NC_PAGED_WAVES, THREADS = 64 * NW;
    // Weights are 2^(score - max) times UNIT, in 16-bit parts. f16: the largest fits, the high part is normal down to 2^-29 of
    // it and the low part, which has a unit of its own (kLowUnit), wherever the high part is: 2^-22 of the weight, or below
    // 2^-29 of the largest one 2^-52 of that. (Both parts in one unit of 2^12 lost all weights below 2^-37, which are what
    // counts where the largest one's V is 0.) bf16: the sum of 2^31 V at the type's largest value (2^128) stays finite, and V
    // below 2^-94 may count as 0; the parts are normal down to 2^-78 of the largest weight. The product with UNIT is exact;
    // added to the exponent (-32 and a score of 2^-24 steps) it took 1.3e-6 of every weight.
    static constexpr float UNIT = BF ? 0x1p-32f : 0x1p15f;
    static constexpr int PARTS = BF ? 3 : 2;
    using KReg = typename std::conditional<D == 16, u32x2, u32x4>::type;
    using VReg = typename std::conditional<FOUR || E <= 2, uint32_t, typename std::conditional<E == 4, u32x2, u32x4>::type>::type;
    using QPart = typename std::conditional<SIXES, u32x6, u32x8>::type;
    using Elem = typename std::conditional<FOUR, uint8_t, uint16_t>::type;
    struct NoScales {};
    // Of V a lane loads one scale of a tile, that of key 4g + c % 4 and its own dims; the lane's four keys' are those of the four
    // lanes next to each other.
    struct Scales {
        uint32_t k[NT], v[NT];
    };

    // K and V of a wave's step, on their way or there, and which keys count: the first seen[t] of a tile, or
    // (pages of any size) those whose bits are set in it.
    struct Step {
        KReg k[NT][KL];
        VReg v[NT][4];
        uint32_t seen[NT];
        typename std::conditional<FOUR, Scales, NoScales>::type scale;
    };
    struct Pages {
        uint32_t e[NT];
    };
    // One request's table row and one key head of the pools. Off: a page fits 32 bits where a tile lies in one.
    using Off = typename std::conditional<UNI, uint32_t, uint64_t>::type;
    struct Cache {
        const int32_t *table;
        const Elem *k, *v;
        const uint8_t *ks, *vs;
        uint64_t values;  // FOUR: of the pool, from there on
        Off page_stride, token_stride;
        uint32_t num_pages;
        nc_paged_div ps;
    };

    const Args args;
    const uint32_t lane, w, c, g;
    const uint32_t wave_shift;
    const uint32_t bk;       // keys of a block
    const uint32_t qt, kw;   // this wave's part of the query heads, and of a block's keys
    float (*s_o)[16][OP];    // [NW]
    float (*s_ml)[16][2];    // [NW]
    uint32_t *s_word;

    uint32_t kat, vat[4];    // byte offsets of the lane's K and V in a tile
    float sc;                // scale * log2(e)
    u32x4 qv[FOUR ? 1 : KK];
    QPart qp[FOUR ? KK : 1];  // FOUR: Q's parts and the bytes of their scales
    uint32_t qs[FOUR ? KK : 1];
    float by;                 // SIXES: sc over what the lane's query was multiplied by
    uint32_t ksat, vsat;      // and byte offsets of the scales
    const uint16_t *q_row;    // the lane's query
    float *score;             // MASS: the lane's row of scores, at its keys of a tile; null for a column without a query
    float *row_ml;            // and the head's (max, 1 / sum)
    floatx4 acc[E];
    float m, l;

    // Blocks of WK * (NW >> shift) keys.
    static __device__ __forceinline__ uint32_t blocks_by(uint32_t len, uint32_t shift) {
        return (len + (WK * NW >> shift) - 1u) >> (__builtin_ctz(WK * NW) - shift);
    }
    __device__ __forceinline__ uint32_t blocks_of(uint32_t len) const { return blocks_by(len, wave_shift); }
    // Query heads of a piece.
    __device__ __forceinline__ uint32_t piece_rows(Args a) const { return NEXT ? a->group << wave_shift : a->rows; }
    static __device__ __forceinline__ uint32_t units_of(uint32_t nb) { return nb ? nb + HEAD_UNITS : 0u; }

    // Q of a block's query heads as the B operand: lane (c, g) holds query c of the wave's 16, dims KE*g.. of 32.
    __device__ __forceinline__ void load_q(uint32_t r, uint32_t head0, uint32_t rows) {
        const Args a = again(args);
        const uint32_t col = c & (COLS - 1u);
        const uint32_t row = NEXT ? qt * a->group + min(col, a->group - 1u) : min(16u * qt + col, rows - 1u);
        const uint16_t *p = a->q + r * a->q_stride + (head0 + row) * a->q_head_stride;
        if constexpr (MASS) {
            const auto more = more_of(a);
            float *s = more->scores + ((uint64_t)r * a->num_q_heads + head0 + row) * more->score_pitch + 4 * g;
            score = (NEXT ? col < a->group : 16u * qt + col < rows) ? s : nullptr;
            row_ml = more->row_ml + 2 * ((uint64_t)r * a->num_q_heads + head0);
        }
        if constexpr (FOUR) {  // loaded in sweep(), behind what it has to wait for longer
            q_row = p;
            return;
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const uint16_t *x = p + 32 * kk + KE * g;
            u32x4 t = {0u, 0u, 0u, 0u};
            if (a->q_vec) {
                if constexpr (D == 16) {
                    const u32x2 y = *reinterpret_cast<const u32x2 *>(x);
                    t[0] = y[0];
                    t[1] = y[1];
                } else {
                    t = *reinterpret_cast<const u32x4 *>(x);
                }
            } else {
#pragma unroll
                for (int i = 0; i < KE / 2; ++i) t[i] = uint32_t(x[2 * i]) | uint32_t(x[2 * i + 1]) << 16;
            }
            qv[kk] = t;
        }
    }

    // The group of 32 dims that the lane holds of a K row.
    __device__ __forceinline__ uint32_t k_group() const { return D == 128 ? g : D == 64 ? g & 1u : 0u; }

    // FOUR: the query's 128 columns are, by 32 that share a scale, D = 128: its dims, once for each part; 64: the dims of parts 0
    // and 1, then of parts 2 and 3; 32: the dims of parts 0 to 3. K's are its dims as often. Lane (c, g) holds the scale of columns 32g..+31,
    // and those columns in 6 bits, in 8 columns 16g..+15 and 64+16g..+15 (hw_probe.hip has the layouts). The parts' scale is
    // the power of two of the largest value of its 32 dims, so that a large channel takes no bits from the others' dims, and what the
    // parts leave is 2^-25 of that at most: nothing of an f16 value above 2^-14 of it, or a bf16 value above 2^-17. (Three e4m3 parts under
    // one scale for the row left 2^-20 of its largest value: with a channel at 256 times the others, scores were off by 1e-4.)
    struct RawQ {
        uint32_t w[QDIMS / 2];
        bool bf;
    };
    __device__ __forceinline__ RawQ load_raw_q() const {
        const Args a = again(args);
        RawQ q;
        q.bf = more_of(a)->bf;
        const uint16_t *x = q_row + QDIMS * (D == 32 ? g & 1u : g);
        if (a->q_vec) {
#pragma unroll
            for (int u = 0; u < QDIMS / 8; ++u) {
                const u32x4 y = *reinterpret_cast<const u32x4 *>(x + 8 * u);
#pragma unroll
                for (int i = 0; i < 4; ++i) q.w[4 * u + i] = y[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < QDIMS / 2; ++i) q.w[i] = uint32_t(x[2 * i]) | uint32_t(x[2 * i + 1]) << 16;
        }
        return q;
    }
    __device__ __forceinline__ void split_q(const RawQ &q) {
        float f[QDIMS];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < QDIMS / 2; ++i) {
            const half2v h = __builtin_bit_cast(half2v, q.w[i]);
            f[2 * i] = q.bf ? __uint_as_float(q.w[i] << 16) : (float)h[0];
            f[2 * i + 1] = q.bf ? __uint_as_float(q.w[i] & 0xffff0000u) : (float)h[1];
            top = max(top, max(__float_as_uint(f[2 * i]) & 0x7fffffffu, __float_as_uint(f[2 * i + 1]) & 0x7fffffffu));
        }
        if constexpr (SIXES)
            split_sixes(f, top >> 23);
        else
            split_eights(f, pair_max(top) >> 23);
    }
    // e: the exponent of the largest of the 32 dims; 255 where one is not finite: so is the scale then.
    __device__ __forceinline__ void split_eights(const float (&f)[QDIMS], uint32_t e) {
        // The last part's scale byte is 1 or more; what is smaller than that allows for still has all of bf16's bits.
        e = max(e, 1u + 5u * (QPARTS - 1));
        u32x4 part[QPARTS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[4] = {f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
#pragma unroll
            for (int n = 0; n < QPARTS; ++n) {
                const float scale = __uint_as_float((e - 5u * n) << 23);
                part[n][i] = n + 1 < QPARTS ? take_eights<false>(x, scale) : take_eights<true>(x, scale);
            }
        }
        uint32_t n = g;  // the part whose scale is the lane's, in the first product
        if constexpr (D == 64) {
            // g = 0, 1 have one 32's exponent and g = 2, 3 the other's; as scales they take turns
            const auto half = __builtin_amdgcn_permlane32_swap(e, e, false, false);
            e = __builtin_amdgcn_permlane16_swap(half[0], half[1], false, false)[0];
            n = g >> 1;
        }
#pragma unroll
        for (int k = 0; k < KK; ++k) {
            const u32x4 x = D == 64 ? part[2 * k] : g < 2 ? part[0] : part[1], y = D == 64 ? part[2 * k + 1] : g < 2 ? part[2] : part[3];
            if constexpr (!SIXES) qp[k] = u32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            qs[k] = e == 255u ? e : e - 5u * (n + 2 * k);
        }
    }
    __device__ __forceinline__ void split_sixes(const float (&f)[QDIMS], uint32_t e) {
        floatx16 x, y;
#pragma unroll
        for (int i = 0; i < QDIMS / 2; ++i) {
            x[i] = f[2 * i];
            y[i] = f[2 * i + 1];
        }
        // The last part's scale byte is 1 or more here too, which leaves up to 2^-130. A query of less than 2^-47 all over (in bf16) is
        // taken 2^32 times as large, at which no product overflows.
        by = sc;
        if (__any(e < 80u)) {
            const bool all = quad_max(e) < 80u;
#pragma unroll
            for (int i = 0; i < QDIMS / 2; ++i) {
                x[i] *= all ? 0x1p32f : 1.f;
                y[i] *= all ? 0x1p32f : 1.f;
            }
            e += all ? 32u : 0u;
            by = all ? sc * 0x1p-32f : sc;
        }
        e = max(e, 2u + 5u * (QPARTS - 1));
#pragma unroll
        for (int n = 0; n < QPARTS; ++n) {
            const float scale = __uint_as_float((e - 1u - 5u * n) << 23);  // of n = 0, the largest is 2 to 4 times that
            const u32x6 w = n + 1 < QPARTS ? take_sixes<false>(x, y, scale) : take_sixes<true>(x, y, scale);
            if constexpr (SIXES) qp[n] = w;
            qs[n] = e == 255u ? e : e - 1u - 5u * n;
        }
    }

    // Table entries of a step's 16-key tiles: uniform where a tile lies in one page, else one per lane (key c
    // of the tile). Past the request's end the last key's entry.
    __device__ __forceinline__ Pages load_pages(const Cache &a, uint32_t k0, uint32_t len) const {
        Pages p;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (UNI)
                p.e[t] = (uint32_t)as_const(a.table)[nc_paged_quot(min(k0 + 16 * t, len - 1u), a.ps)];
            else
                p.e[t] = (uint32_t)a.table[nc_paged_quot(min(k0 + 16 * t + c, len - 1u), a.ps)];
        }
        return p;
    }

    // Sets the loads of the keys k0..k0+WK-1 of one key head under way, those below `end`.
    // UNI: a tile is a buffer of its own whose length ends with its last key that counts, so that what lies
    // behind is neither read nor waited for, and is 0. Else rows that do not count read the pool's first row.
    __device__ __forceinline__ void issue(Step &st, const Cache &a, const Pages &pages, uint32_t k0, uint32_t end) const {
        if constexpr (UNI) {
            const uint32_t ts = 2u * a.token_stride;
            __amdgpu_buffer_rsrc_t vb[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t k1 = k0 + 16 * t;
                const bool in = k1 < end && pages.e[t] < a.num_pages;
                const uint32_t n = in ? min(end - k1, 16u) : 0u;
                st.seen[t] = n;
                const uint32_t tok = k1 - nc_paged_quot(k1, a.ps) * a.ps.d;
                const uint64_t at = in ? (uint64_t)pages.e[t] * a.page_stride + tok * a.token_stride : 0u;
                const __amdgpu_buffer_rsrc_t kb = tile(a.k + at, n * ts);
                vb[t] = tile(a.v + at, n * ts);
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    if constexpr (D == 16)
                        st.k[t][kk] = __builtin_amdgcn_raw_buffer_load_b64(kb, kat, 0, 0);
                    else
                        st.k[t][kk] = __builtin_amdgcn_raw_buffer_load_b128(kb, kat + 64 * kk, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (E == 8)
                        st.v[t][i] = __builtin_amdgcn_raw_buffer_load_b128(vb[t], vat[i], 0, 0);
                    else if constexpr (E == 4)
                        st.v[t][i] = __builtin_amdgcn_raw_buffer_load_b64(vb[t], vat[i], 0, 0);
                    else if constexpr (E == 2)
                        st.v[t][i] = __builtin_amdgcn_raw_buffer_load_b32(vb[t], vat[i], 0, 0);
                    else
                        st.v[t][i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vb[t], vat[i], 0, 0);
                }
        } else {
            const uint16_t *vb[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t key = k0 + 16 * t + c;
                const bool in = key < end && pages.e[t] < a.num_pages;
                st.seen[t] = (uint32_t)__ballot(in) & 0xffffu;
                const uint64_t at = in ? pages.e[t] * a.page_stride + (key - nc_paged_quot(key, a.ps) * a.ps.d) * a.token_stride : 0u;
                const uint16_t *kp = a.k + at + KE * g;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) st.k[t][kk] = *reinterpret_cast<const KReg *>(kp + 32 * kk);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int from = 4 * (int)g + i;
                    const uint32_t lo = __shfl((uint32_t)at, from, 64), hi = __shfl((uint32_t)(at >> 32), from, 64);
                    vb[t][i] = a.v + ((uint64_t)hi << 32 | lo) + E * c;
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (E > 1)
                        st.v[t][i] = *reinterpret_cast<const VReg *>(vb[t][i]);
                    else
                        st.v[t][i] = *vb[t][i];
                }
        }
    }

    // The same of a 4-bit cache where a tile lies in one page: `at` has, by lane, the places of NT tiles of as many steps as there are
    // lanes for, in units of 32 values (all ones: on no page, or past the end); these are the tiles of step `n`. A pool is one
    // buffer, whose bytes 32 bits can count; rows that do not count are read too.
    __device__ __forceinline__ void issue_tiles(Step &st, const Cache &a, uint32_t places, uint32_t n, uint32_t k0, uint32_t end) const {
        const uint32_t codes = (uint32_t)(a.values / 2u), scales = (uint32_t)(a.values / 32u);
        const __amdgpu_buffer_rsrc_t kb = tile(a.k, codes), vb = tile(a.v, codes), ks = tile(a.ks, scales), vs = tile(a.vs, scales);
        uint32_t at[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            at[t] = __builtin_amdgcn_readlane(places, NT * n + t);
            const bool in = at[t] != ~0u;
            st.seen[t] = in ? min(end - (k0 + 16 * t), 16u) : 0u;
            at[t] = in ? at[t] : 0u;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            st.k[t][0] = __builtin_amdgcn_raw_buffer_load_b128(kb, kat, 16u * at[t], 0);
            st.scale.k[t] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(ks, ksat, at[t], 0);
            st.scale.v[t] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(vs, vsat, at[t], 0);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (E == 8)
                    st.v[t][i] = __builtin_amdgcn_raw_buffer_load_b32(vb, vat[i], 16u * at[t], 0);
                else if constexpr (E == 4)
                    st.v[t][i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vb, vat[i], 16u * at[t], 0);
                else
                    st.v[t][i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(vb, vat[i], 16u * at[t], 0);
            }
    }

    // On pages of any size: lane j has the place of key j of the step, as above.
    __device__ __forceinline__ void issue_keys(Step &st, const Cache &a, uint32_t places, uint32_t k0) const {
        const uint64_t here = __ballot(places != ~0u);
        places = places != ~0u ? places : 0u;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            st.seen[t] = (uint32_t)(here >> (16 * t)) & 0xffffu;
            const uint64_t at = (uint32_t)__shfl((int)places, 16 * t + (int)c, 64);
            st.k[t][0] = *reinterpret_cast<const u32x4 *>(a.k + 16u * at + 16u * k_group());
            st.scale.k[t] = a.ks[at + k_group()];
            const uint64_t vat = (uint32_t)__shfl((int)places, 16 * t + 4 * (int)g + (int)(c % 4u), 64);
            st.scale.v[t] = a.vs[vat + E * c / 32u];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t at = (uint32_t)__shfl((int)places, 16 * t + 4 * (int)g + i, 64);
                const uint8_t *x = a.v + 16u * at + E / 2 * c;
                if constexpr (E == 8)
                    st.v[t][i] = *reinterpret_cast<const uint32_t *>(x);
                else if constexpr (E == 4)
                    st.v[t][i] = *reinterpret_cast<const uint16_t *>(x);
                else
                    st.v[t][i] = *x;
            }
    }

    // The steps of sweep() over such a cache; the table's entries a step ahead.
    __device__ __forceinline__ void sweep_keys(const Cache &a, uint32_t k0, uint32_t end, uint32_t by) {
        static_assert(WK == 64 || !FOUR, "a key a lane");
        auto entry_of = [&](uint32_t from) {
            const uint32_t key = from + lane;
            return key < end ? (uint32_t)a.table[nc_paged_quot(key, a.ps)] : ~0u;
        };
        auto place_of = [&](uint32_t from, uint32_t entry) {
            const uint32_t key = from + lane;
            return entry < a.num_pages ? (uint32_t)((entry * a.page_stride + (key - nc_paged_quot(key, a.ps) * a.ps.d) * a.token_stride) / 32u) : ~0u;
        };
        uint32_t entry = entry_of(k0);
        const RawQ q = load_raw_q();
        Step x;
        issue_keys(x, a, place_of(k0, entry), k0);
        entry = entry_of(k0 + by);
        split_q(q);
        while (true) {
            compute(x, k0, end);
            if ((k0 += by) >= end) return;
            issue_keys(x, a, place_of(k0, entry), k0);
            entry = entry_of(k0 + by);
        }
    }

    // The steps of sweep() over a 4-bit cache whose tiles lie in one page each. The table's entries are read 64 / NT steps at a time,
    // that many steps ahead: as scalar loads, one after the other, they took a third of a step. Q's loads are under way beside the
    // first entries', and it is split while the first step's are. (With one place in the code for a step's loads, and that split
    // behind a branch, long requests took 8 % longer and short ones 2 % less.)
    __device__ __forceinline__ void sweep_tiles(const Cache &a, uint32_t k0, uint32_t end, uint32_t by) {
        constexpr uint32_t STEPS = 64 / NT;
        const uint32_t mine = lane / NT * by + 16u * (lane % NT);  // the lane's tile, behind the batch's first key
        auto entry_of = [&](uint32_t from) {
            const uint32_t key = from + mine;
            return key < end ? (uint32_t)a.table[nc_paged_quot(key, a.ps)] : ~0u;
        };
        auto place_of = [&](uint32_t from, uint32_t entry) {
            const uint32_t key = from + mine;
            return entry < a.num_pages ? (entry * a.page_stride + (key - nc_paged_quot(key, a.ps) * a.ps.d) * a.token_stride) / 32u : ~0u;
        };
        uint32_t batch = k0, n = 0, entry = entry_of(k0);
        const RawQ q = load_raw_q();
        uint32_t places = place_of(k0, entry);
        auto next = [&](Step &st, uint32_t key) {
            if (n == STEPS) {
                batch += STEPS * by;
                places = place_of(batch, entry);
                entry = entry_of(batch + STEPS * by);
                n = 0;
            }
            issue_tiles(st, a, places, n++, key, end);
        };
        Step x;
        next(x, k0);
        entry = entry_of(k0 + STEPS * by);
        split_q(q);
        while (true) {
            compute(x, k0, end);
            if ((k0 += by) >= end) return;
            next(x, k0);
        }
    }

    // A raw buffer of `bytes` bytes.
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(const Elem *p, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<Elem *>(p), 0, (int)bytes, 0x00020000);
    }

    static __device__ __forceinline__ uint32_t word(const VReg &v, int i) {
        if constexpr (E > 2 && !FOUR)
            return v[i];
        else
            return v;
    }

    // What lane j of each 4 has.
    static __device__ __forceinline__ float v_scale(uint32_t x, int j) {
        switch (j) {
            case 0: return __uint_as_float(__builtin_amdgcn_update_dpp(0, x, 0x00, 0xf, 0xf, true));  // quad_perm j,j,j,j
            case 1: return __uint_as_float(__builtin_amdgcn_update_dpp(0, x, 0x55, 0xf, 0xf, true));
            case 2: return __uint_as_float(__builtin_amdgcn_update_dpp(0, x, 0xaa, 0xf, 0xf, true));
            default: return __uint_as_float(__builtin_amdgcn_update_dpp(0, x, 0xff, 0xf, 0xf, true));
        }
    }

    // V's dims 2i, 2i+1 of key j of tile t.
    static __device__ __forceinline__ uint32_t v_pair(const Step &st, int t, int j, int i) {
        if constexpr (FOUR)
            return pair_of_fours(st.v[t][j], v_scale(st.scale.v[t] << 23, j), i);
        else
            return word(st.v[t][j], i);
    }

    // k0: the first key, of those below `end`.
    __device__ __forceinline__ void compute(Step &st, uint32_t k0, uint32_t end) {
        bool full = true;
#pragma unroll
        for (int t = 0; t < NT; ++t) full = full && st.seen[t] == (UNI ? 16u : 0xffffu);
        float s[SETS][4];
        float top = neg_inf();
        floatx4 dot[NT];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const floatx4 x = kk ? dot[t] : floatx4{0.f, 0.f, 0.f, 0.f};
                if constexpr (FOUR) {
                    const i32x4 y = __builtin_bit_cast(i32x4, st.k[t][0]);
                    i32x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < (SIXES ? 6 : 8); ++i) z[i] = (int)qp[kk][i];
                    dot[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(i32x8{y[0], y[1], y[2], y[3], 0, 0, 0, 0}, z, x, 4, SIXES ? 2 : 0, 0,
                                                                             (int)st.scale.k[t], 0, (int)qs[kk]);
                } else if constexpr (D == 16)
                    dot[t] = mfma_k16<BF>(st.k[t][kk], u32x2{qv[kk][0], qv[kk][1]}, x);
                else
                    dot[t] = mfma_k32<BF>(st.k[t][kk], qv[kk], x);
            }
        const uint32_t part = c / COLS;  // the column group
#pragma unroll
        for (int t = 0; t < SETS; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = dot[PACK * t][i];
#pragma unroll
                for (int n = 1; n < PACK; ++n) x = part == (uint32_t)n ? dot[PACK * t + n][i] : x;
                s[t][i] = x * (FOUR && SIXES ? by : sc);
            }
        if (!full) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = UNI ? 4 * g + i < st.seen[t] : st.seen[t] >> (4 * g + i) & 1u;
                    if (PACK == 1 || part == (uint32_t)(t % PACK)) s[t / PACK][i] = in ? s[t / PACK][i] : neg_inf();
                    if constexpr (!FOUR && !UNI) {  // 0 * NaN would be NaN
                        if constexpr (E > 2) {
#pragma unroll
                            for (int j = 0; j < E / 2; ++j) st.v[t][i][j] = in ? st.v[t][i][j] : 0u;
                        } else {
                            st.v[t][i] = in ? st.v[t][i] : 0u;
                        }
                    }
                }
                if constexpr (FOUR) {
                    const uint32_t key = 4 * g + c % 4u;
                    if (UNI ? key >= st.seen[t] : !(st.seen[t] >> key & 1u)) st.scale.v[t] = 0u;
                }
            }
        }
        if constexpr (MASS) {  // a row holds whole tiles; keys that do not count have -infinity
            if (score) {
#pragma unroll
                for (int t = 0; t < SETS; ++t) {
                    const uint32_t at = k0 + 16 * (PACK * t + part);
                    if (at < end) *reinterpret_cast<floatx4 *>(score + at) = floatx4{s[t][0], s[t][1], s[t][2], s[t][3]};
                }
            }
        }
#pragma unroll
        for (int t = 0; t < SETS; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
        top = fmaxf(m, quad_max(top));
        const float ref = finite_or_0(top);
        if (!__all(top == m)) {
            const float f = __builtin_amdgcn_exp2f(m - ref);
            l *= f;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] *= f;
            m = top;
        }
#pragma unroll
        for (int t = 0; t < SETS; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - ref) * UNIT;
                l += s[t][i];
            }
        u32x4 p[KT][PARTS];
        if constexpr (PACK == 1) {
#pragma unroll
            for (int u = 0; u < KT; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int n = 0; n < PARTS; ++n)
                        p[u][n][j] = take_pair<BF, FOUR>(s[2 * u + j / 2][2 * (j % 2)], s[2 * u + j / 2][2 * (j % 2) + 1]);
        } else {  // a column group's weights stand at its own tile's keys, the others' are 0
#pragma unroll
            for (int t = 0; t < SETS; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int n = 0; n < PARTS; ++n) {
                        const uint32_t w = take_pair<BF, FOUR>(s[t][2 * j], s[t][2 * j + 1]);
#pragma unroll
                        for (int x = 0; x < PACK; ++x) {
                            const int at = PACK * t + x;  // the tile
                            p[at / 2][n][2 * (at % 2) + j] = part == (uint32_t)x ? w : 0u;
                        }
                    }
        }
        constexpr int G = E < 2 ? E : 2;  // products of so many dims in turn: each waits for its last one
#pragma unroll
        for (int i0 = 0; i0 < E; i0 += G) {
            floatx4 low[G];  // the lower parts' products
#pragma unroll
            for (int i = 0; i < G; ++i) low[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < KT; ++u) {
                u32x4 x[G];
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t lo = v_pair(st, 2 * u + j / 2, 2 * (j % 2), (i0 + i) / 2);
                        const uint32_t hi = v_pair(st, 2 * u + j / 2, 2 * (j % 2) + 1, (i0 + i) / 2);
                        x[i][j] = __builtin_amdgcn_perm(hi, lo, i % 2 ? 0x07060302u : 0x05040100u);
                    }
#pragma unroll
                for (int n = 0; n < PARTS; ++n)
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        floatx4 &sum = n && !FOUR ? low[i] : acc[i0 + i];
                        sum = mfma_k32<BF>(x[i], p[u][n], sum);
                    }
            }
            if constexpr (FOUR) continue;  // whose V are finite, or NaN
            // An infinite V times a lower part, which may be 0 or negative, must not undo what its high part gave: no such
            // sum of finite V comes near 2^100.
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i0 + i][j] = __builtin_fmaf(__builtin_amdgcn_fmed3f(low[i][j], -0x1p100f, 0x1p100f), BF ? 1.f : 1.f / kLowUnit, acc[i0 + i][j]);
        }
    }

    // The keys k0, k0 + by, ... below `end` of one key head: AHEAD, a step's loads are under way before the step before
    // it is computed, and the table entries a step earlier. Every step's loads are the same ones whatever there
    // is to load, so that waiting for one step's does not mean waiting for the next step's too.
    __device__ __forceinline__ void sweep(uint32_t r, uint32_t kvh, uint32_t k0, uint32_t end, uint32_t len, uint32_t by) {
        if (k0 >= end) return;
        const Args a = again(args);
        Cache cache;
        cache.table = a->table + r * a->table_stride;
        if constexpr (FOUR) {
            const auto more = more_of(a);
            const uint64_t at = kvh * a->head_stride;
            cache.k = reinterpret_cast<const uint8_t *>(a->k) + at / 2;
            cache.v = reinterpret_cast<const uint8_t *>(a->v) + at / 2;
            cache.ks = more->k_scales + at / 32;
            cache.vs = more->v_scales + at / 32;
            cache.values = more->values - at;
        } else {
            cache.k = a->k + kvh * a->head_stride;
            cache.v = a->v + kvh * a->head_stride;
        }
        cache.page_stride = a->page_stride;
        cache.token_stride = a->token_stride;
        cache.num_pages = a->num_pages;
        cache.ps.d = a->ps.d;
        cache.ps.magic = a->ps.magic;
        cache.ps.shift = a->ps.shift;
        if constexpr (FOUR && UNI)
            sweep_tiles(cache, k0, end, by);
        else if constexpr (FOUR)
            sweep_keys(cache, k0, end, by);
        else
            sweep_steps(cache, k0, end, len, by);
    }

    __device__ __forceinline__ void sweep_steps(const Cache &cache, uint32_t k0, uint32_t end, uint32_t len, uint32_t by) {
        Step x, y;
        Pages pages = load_pages(cache, k0, len);
        issue(x, cache, pages, k0, end);
        if constexpr (!AHEAD) {
            while (true) {
                pages = load_pages(cache, k0 + by, len);
                compute(x, k0, end);
                if ((k0 += by) >= end) return;
                issue(x, cache, pages, k0, end);
            }
        }
        if (k0 + by >= end) {
            compute(x, k0, end);
            return;
        }
        pages = load_pages(cache, k0 + by, len);
        while (true) {
            issue(y, cache, pages, k0 + by, end);
            pages = load_pages(cache, k0 + 2 * by, len);
            compute(x, k0, end);
            if (k0 + by >= end) break;
            issue(x, cache, pages, k0 + 2 * by, end);
            pages = load_pages(cache, k0 + 3 * by, len);
            compute(y, k0 + by, end);
            k0 += 2 * by;
            if (k0 >= end) break;
        }
    }

    // Row q of the piece of workgroup j, `first` of which began the request and head.
    static __device__ __forceinline__ uint64_t piece_row(uint32_t j, uint32_t first, uint32_t piece_rows, uint32_t q) {
        return ((uint64_t)j * 2 + (j == first)) * piece_rows + q;
    }

    static __device__ __forceinline__ floatx4 get4(const float *p) {
        float p0, p1, p2, p3;
        get2(p, p0, p1);
        get2(p + 2, p2, p3);
        return floatx4{p0, p1, p2, p3};
    }

    // Up to N pieces, which are all: every thread has their maxima and sums with its columns, in one go.
    template <uint32_t N>
    __device__ __forceinline__ void merge_few(uint32_t lead, uint32_t stride, uint32_t count, uint32_t first, uint32_t rows, float *o) {
        const Args a = again(args);
        const float *part_ml = a->part_ml, *part_o = a->part_o;
        const uint32_t per_piece = piece_rows(a);
        for (uint32_t it = threadIdx.x; it < rows * (D / 4); it += THREADS) {
            const uint32_t q = it / (D / 4), x = 4 * (it % (D / 4));
            float pm[N], pl[N], top = neg_inf(), sum = 0.f;
            floatx4 po[N], out = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t n = 0; n < N; ++n) {
                const uint64_t at = piece_row(lead + min(n, count - 1u) * stride, first, per_piece, q);
                get2(part_ml + 2 * at, pm[n], pl[n]);
                po[n] = get4(part_o + at * D + x);
            }
#pragma unroll
            for (uint32_t n = 0; n < N; ++n) top = fmaxf(top, pm[n]);
#pragma unroll
            for (uint32_t n = 0; n < N; ++n)
                if (n < count) {
                    const float f = __builtin_amdgcn_exp2f(pm[n] - finite_or_0(top));
                    sum += f * pl[n];
                    out += f * po[n];
                }
            store_o(o, q, x, out, sum, top);
        }
    }

    // Adds `count` pieces of one request and head, those of workgroups lead, lead + stride, ..., in their order: to O if
    // there are no others, else in the place of the first of them. Their maxima, a piece a lane, give every piece's
    // factor, kept in LDS; the first pieces of O are on their way meanwhile. Four columns of a row are a thread's;
    // where that leaves threads over, groups of them take every so many-th piece.
    __device__ __forceinline__ void merge(uint32_t lead, uint32_t stride, uint32_t count, uint32_t first, bool all, uint32_t rows, float *o) {
        constexpr uint32_t PF = 4;
        const Args a = again(args);
        const uint32_t items = rows * (D / 4), per_piece = piece_rows(a);
        const uint32_t groups = items > THREADS / 2 ? 1u : min(THREADS / items, (count - 1u) / PF + 1u);
        float *part_ml = a->part_ml, *part_o = a->part_o;
        float *s_f = &s_o[0][0][0], *s_tot = s_f + NC_PAGED_MERGE_ROWS;
        floatx4 *s_sum = reinterpret_cast<floatx4 *>(s_tot + 2 * 64);
        const uint32_t grp = groups == 1 ? 0u : threadIdx.x / items;
        const bool works = grp < groups;
        uint32_t it = threadIdx.x - grp * items;
        floatx4 po[PF];
        auto load = [&](uint32_t n0) {
            const uint32_t q = it / (D / 4), x = 4 * (it % (D / 4));
#pragma unroll
            for (uint32_t n = 0; n < PF; ++n)
                po[n] = get4(part_o + piece_row(lead + min(n0 + n * groups, count - 1u) * stride, first, per_piece, q) * D + x);
        };
        if (works && it < items) load(grp);
        const uint32_t lanes = count > 16u ? 6u : count > 4u ? 4u : 2u;  // log2 of a row's
        const uint32_t per = 64u >> lanes;                                // rows of a wave at a time
        for (uint32_t q0 = w * per; q0 < rows; q0 += NW * per) {
            const uint32_t n = lane & ((1u << lanes) - 1u), q = q0 + (lane >> lanes);
            float pm = neg_inf(), pl = 0.f;
            if (n < count && q < rows) get2(part_ml + 2 * piece_row(lead + n * stride, first, per_piece, q), pm, pl);
            float top = near<true>(pm, lanes > 2u);
            if (lanes > 4u) top = quad_max(top);
            const float f = __builtin_amdgcn_exp2f(pm - finite_or_0(top));
            float sum = near<false>(f * pl, lanes > 2u);
            if (lanes > 4u) sum = quad_sum(sum);
            if (n < count && q < rows) s_f[n * rows + q] = f;
            if (n == 0 && q < rows) {
                s_tot[2 * q] = top;
                s_tot[2 * q + 1] = sum;
            }
        }
        __syncthreads();
        for (bool next = false; it < items || groups > 1; it += THREADS, next = true) {
            const uint32_t q = it / (D / 4), x = 4 * (it % (D / 4));
            floatx4 out = {0.f, 0.f, 0.f, 0.f};
            if (works && it < items) {
                for (uint32_t n0 = grp; n0 < count; n0 += PF * groups) {
                    if (next || n0 != grp) load(n0);
#pragma unroll
                    for (uint32_t n = 0; n < PF; ++n)
                        if (n0 + n * groups < count) out += s_f[(n0 + n * groups) * rows + q] * po[n];
                }
            }
            if (groups > 1) {
                s_sum[threadIdx.x] = out;
                __syncthreads();
                if (grp == 0)
                    for (uint32_t n = 1; n < groups; ++n) out += s_sum[threadIdx.x + n * items];
            }
            if (grp == 0 && it < items) {
                if (all) {
                    store_o(o, q, x, out, s_tot[2 * q + 1], s_tot[2 * q]);
                } else {
                    const uint64_t at = piece_row(lead, first, per_piece, q);
                    put2(part_o + at * D + x, out[0], out[1]);
                    put2(part_o + at * D + x + 2, out[2], out[3]);
                    if (x == 0) put2(part_ml + 2 * at, s_tot[2 * q], s_tot[2 * q + 1]);
                }
            }
            if (groups > 1) break;
        }
    }

    // After workgroup i's piece of a request and head whose pieces are those of workgroups first..last: the last
    // of every `fan` to arrive adds theirs up, and the last of those that did, until there is one. A CU reads pieces at a
    // few ten GB/s: one that adds up all 256 of a long request took longer than its keys.
    __device__ __forceinline__ void join(uint32_t i, uint32_t first, uint32_t last, uint32_t rows, float *o) {
        const Args a = again(args);
        const uint32_t pieces = last - first + 1u, per_piece = piece_rows(a);
        const uint32_t fan = nc_paged_one_round(pieces, per_piece * D) ? pieces : nc_paged_fan(per_piece, D);
        uint32_t *counters = a->counters;
        uint32_t c = i - first;
        for (uint32_t stride = 1;; stride *= fan) {
            // Every thread's stores have arrived before the count says so, and pieces are read only after the count
            // showed the last of them.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            c -= c % (fan * stride);
            const uint32_t lead = first + c, count = min(fan, (pieces - c - 1u) / stride + 1u);
            uint32_t *counter = counters + 2 * lead + (lead == first);
            if (threadIdx.x == 0) {
                const uint32_t before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (before == count - 1u) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                *s_word = before;
            }
            __syncthreads();
            if (*s_word != count - 1u) return;
            const bool all = pieces <= fan * stride;
            if (all && count <= 4u)
                merge_few<4>(lead, stride, count, first, rows, o);
            else if (all && count <= 8u)
                merge_few<8>(lead, stride, count, first, rows, o);
            else
                merge(lead, stride, count, first, all, rows, o);
            if (all) return;
            counters += 2 * NC_PAGED_MAX_WGS;  // of the next round
        }
    }

    // What the weights' kernel needs of row q's sum.
    __device__ __forceinline__ void put_ml(uint32_t q, float top, float sum) const {
        row_ml[2 * q] = finite_or_0(top);
        row_ml[2 * q + 1] = sum == 0.f ? 0.f : __builtin_amdgcn_rcpf(sum) * UNIT;
    }

    __device__ __forceinline__ void store_o(float *o, uint32_t q, uint32_t x, floatx4 v, float sum, float top) {
        const float inv = __builtin_amdgcn_rcpf(sum);  // to an ulp
        if constexpr (MASS) {
            if (x == 0) put_ml(q, top, sum);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = sum == 0.f ? 0.f : v[i] * inv;
        const Args a = args;
        float *p = o + q * a->o_head_stride + x;
        if (a->o_vec) {
            *reinterpret_cast<floatx4 *>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = v[i];
        }
    }

    // The column groups' (m, l, O) as one, which all of them get.
    __device__ __forceinline__ void join_columns() {
        if constexpr (PACK > 1) {
            auto add = [](float u, float v) { return u + v; };
            auto over = [](float x, auto &&f) {
                if constexpr (PACK == 4) x = f(x, dpp<0x124>(x));  // row_ror:4 and 8
                return f(x, dpp<0x128>(x));
            };
            const float top = over(m, [](float u, float v) { return fmaxf(u, v); });
            const float f = __builtin_amdgcn_exp2f(m - finite_or_0(top));
            m = top;
            l = over(f * l, add);
#pragma unroll
            for (int i = 0; i < E; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = over(f * acc[i][j], add);
        }
    }

    // O of a head that the wave had to itself: lane (c, g) has dims 4gE..4gE+4E-1 of query c.
    __device__ __forceinline__ void finish_wave(uint32_t r, uint32_t head0, uint32_t rows) {
        const Args a = again(args);
        join_columns();
        const float sum = quad_sum(l);
        if (c >= rows) return;
        if constexpr (MASS) {
            if (g == 0) put_ml(c, m, sum);
        }
        float *o = a->o + r * a->o_stride + head0 * a->o_head_stride;
        const float inv = __builtin_amdgcn_rcpf(sum);  // to an ulp
        o += c * a->o_head_stride + 4 * E * g;
        float v[4 * E];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int j = 0; j < E; ++j) v[x * E + j] = sum == 0.f ? 0.f : acc[j][x] * inv;
#pragma unroll
        for (int x = 0; x < E; ++x) *reinterpret_cast<floatx4 *>(o + 4 * x) = floatx4{v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]};
    }

    // The four waves' (m, l, O) of one run of blocks: to O if the run is all of the request's, else to this
    // workgroup's (i's) piece, to be joined with those of the workgroups that share the units b_lo..b_lo+nb-1, `each`
    // apiece.
    __device__ __forceinline__ void finish(uint32_t rows, uint32_t r, uint32_t head0, bool whole, uint32_t i, uint32_t b_lo, uint32_t nb, uint32_t each) {
        const Args a = again(args);
        uint32_t first = i, last = i;
        if (!whole) {
            first = b_lo / each;
            last = (b_lo + nb - 1u) / each;
        }
        float *o = a->o + r * a->o_stride + head0 * a->o_head_stride;
        join_columns();
        const float sum = quad_sum(l);
        if (g == 0) {
            s_ml[w][c][0] = m;
            s_ml[w][c][1] = sum;
        }
        if (NEXT ? c < a->group : 16 * qt + c < rows) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < E; ++j) s_o[w][c][(4 * g + r) * E + j] = acc[j][r];
        }
        __syncthreads();
        const uint32_t items = rows * (D / 4);
        for (uint32_t it = threadIdx.x; it < items; it += THREADS) {
            const uint32_t q = it / (D / 4), x = 4 * (it % (D / 4));
            // waves q/16 (NEXT: q/group), that + 2^wave_shift, ... hold query q
            const uint32_t j0 = NEXT ? q * a->group_inverse >> 16 : q >> 4, qc = NEXT ? q - j0 * a->group : q & 15u;
            float wm[NW], wl[NW], top = neg_inf(), lsum = 0.f;
            floatx4 wo[NW], out = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t n = 0; n < NW; ++n) {
                const uint32_t j = (j0 + (n << wave_shift)) & (NW - 1u);
                wm[n] = n < NW >> wave_shift ? s_ml[j][qc][0] : neg_inf();
                wl[n] = s_ml[j][qc][1];
                wo[n] = *reinterpret_cast<const floatx4 *>(&s_o[j][qc][x]);
                top = fmaxf(top, wm[n]);
            }
#pragma unroll
            for (uint32_t n = 0; n < NW; ++n) {
                const float f = __builtin_amdgcn_exp2f(wm[n] - finite_or_0(top));
                if (n < NW >> wave_shift) {
                    lsum += f * wl[n];
                    out += f * wo[n];
                }
            }
            if (whole) {
                store_o(o, q, x, out, lsum, top);
            } else {
                const uint64_t at = piece_row(i, first, piece_rows(a), q);
                put2(a->part_o + at * D + x, out[0], out[1]);
                put2(a->part_o + at * D + x + 2, out[2], out[3]);
                if (x == 0) put2(a->part_ml + 2 * at, top, lsum);
            }
        }
        if (!whole) join(i, first, last, rows, o);
        __syncthreads();  // LDS is free again
    }

    // scale: of the scores, in bits. mine: units of this lane's requests; some: how many of them have keys; len0: the length of
    // the last; zero_len: the length of request blockIdx.x.
    __device__ __forceinline__ void run(float scale, uint32_t mine, uint32_t some, uint32_t len0, int32_t zero_len) {
        sc = scale;
        const Args a = args;
        const int32_t *lens = a->seq_lens;
        const uint32_t max_tokens = a->max_tokens;
        const uint32_t R = a->num_seqs, per = (R + 63u) / 64u;  // requests of a lane
        const uint32_t zero_r = blockIdx.x;
        if constexpr (FOUR) {
            const uint32_t ts = (uint32_t)a->token_stride / 2u, ss = (uint32_t)a->token_stride / 32u;
            kat = c * ts + 16u * k_group();
            ksat = c * ss + k_group();
            vsat = (4 * g + c % 4u) * ss + E * c / 32u;
#pragma unroll
            for (int i = 0; i < 4; ++i) vat[i] = (4 * g + i) * ts + E / 2 * c;
        } else {
            kat = 2u * (c * (uint32_t)a->token_stride + KE * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) vat[i] = 2u * ((4 * g + i) * (uint32_t)a->token_stride + E * c);
        }
        const uint32_t incl = wave_scan32(mine), heads = NEXT ? a->heads.d >> wave_shift : a->heads.d;
        const uint32_t total = __builtin_amdgcn_readlane(incl, 63), with_keys = __builtin_amdgcn_readlane(wave_scan32(some), 63);
        const uint32_t units = total * heads, i = blockIdx.x;
        // Heads of many blocks: half the workgroups, which leaves half the pieces to join; one with its loads under way
        // a step ahead keeps a CU's share of the memory busy. Heads of few: the others hide each head's beginning and end.
        const uint32_t most_log2 = total >= NC_PAGED_LONG_UNITS * with_keys ? a->long_log2 : a->short_log2;
        const uint32_t each = nc_paged_each(units, most_log2, NEXT ? 1u : a->each_least), u0 = i * each, u1 = min(u0 + each, units);
        if (u0 < units) {
            // Request r, of length len, whose units begin behind `pre` of the requests before it (times the heads).
            uint32_t r, len, pre;
            {
                // the same request's unit if it had one head
                const uint32_t t = nc_paged_quot(u0, nc_paged_div_by({a->heads.d, a->heads.magic, a->heads.shift}, NEXT ? wave_shift : 0u));
                const uint32_t from = __builtin_ctzll(__ballot(incl - mine <= t && t < incl));
                pre = __builtin_amdgcn_readlane(incl - mine, from);
                r = from * per;
                len = __builtin_amdgcn_readlane(len0, from);
                if (per > 1) {
                    const uint32_t r0 = r, most = min(per, R - r0);
                    for (uint32_t x = 0; x < most; x += 64) {
                        const uint32_t n = x + lane < most ? nc_paged_cut(lens[r0 + x + lane], max_tokens) : 0u;
                        const uint32_t un = units_of(blocks_of(n)), sc = wave_scan32(un);
                        const uint64_t hit = __ballot(t < pre + sc);
                        if (hit) {
                            const uint32_t y = __builtin_ctzll(hit);
                            r = r0 + x + y;
                            len = __builtin_amdgcn_readlane(n, y);
                            pre += __builtin_amdgcn_readlane(sc - un, y);
                            break;
                        }
                        pre += __builtin_amdgcn_readlane(sc, 63);
                    }
                }
                pre *= heads;
            }
            uint32_t nb = blocks_of(len), head = heads > 1 ? (u0 - pre) / units_of(nb) : 0u, seg = pre + head * units_of(nb);
            while (seg < u1) {  // the head's units: its own cost, then one per block
                const bool short_head = nb <= NC_PAGED_WHOLE_BLOCKS;
                const uint32_t b_lo = seg + HEAD_UNITS;  // unit of block 0
                uint32_t b0 = u0 > b_lo ? u0 - b_lo : 0u, b1 = u1 > b_lo ? min(nb, u1 - b_lo) : 0u;
                if (short_head) {  // all of it is the workgroup's that has its first unit
                    b0 = 0;
                    b1 = seg >= u0 ? nb : 0u;
                }
                // Short heads of a request in a row, whose first units are here: a wave each if that takes no more steps than
                // there are heads.
                uint32_t n = 1;
                if constexpr (MANY) {
                    if (nb == 1 && seg >= u0 && a->many && (!NEXT || wave_shift == 0)) {
                        n = min(min(heads - head, NW), (u1 - seg + units_of(1) - 1u) / units_of(1));
                        if (len > n * WK) n = 1;
                    }
                }
                const bool alone = MANY && n > 1;
                if (alone ? w < n : b0 < b1) {
                    uint32_t kvh = alone ? head + w : head, part = 0;
                    if constexpr (NEXT) {
                        if (!alone) kvh = (head << wave_shift) + qt;
                    } else if (a->head_parts > 1) {
                        kvh = head / a->head_parts;
                        part = head - kvh * a->head_parts;
                    }
                    const uint32_t rows = NEXT ? piece_rows(a) : min(64u, a->group - 64u * part);
                    const uint32_t head0 = NEXT ? (alone ? kvh : head) * rows : kvh * a->group + 64u * part;
                    load_q(r, head0, rows);
                    m = neg_inf();
                    l = 0.f;
#pragma unroll
                    for (int x = 0; x < E; ++x) acc[x] = floatx4{0.f, 0.f, 0.f, 0.f};
                    sweep(r, kvh, alone ? 0 : b0 * bk + kw * WK, alone ? len : min(b1 * bk, len), len, alone ? WK : bk);
                    if (alone)
                        finish_wave(r, head0, rows);
                    else
                        finish(rows, r, head0, b0 == 0 && b1 == nb, i, b_lo, nb, each);
                }
                seg += n * units_of(nb);
                if (seg >= u1) break;
                if ((head += n) == heads) {
                    head = 0;
                    // The next request with keys: the next one, or behind empty ones 64 at a time (one by one, and to the end
                    // where there was none, a batch of 4096 of which only the first had keys took 271 us).
                    len = ++r < R ? nc_paged_cut(as_const(lens)[r], max_tokens) : 0u;
                    for (uint32_t r0 = r + 1u; len == 0 && r0 < R; r0 += 64) {
                        const uint32_t x = r0 + lane < R ? nc_paged_cut(lens[r0 + lane], max_tokens) : 0u;
                        const uint64_t hit = __ballot(x != 0);
                        if (hit) {
                            const uint32_t y = __builtin_ctzll(hit);
                            r = r0 + y;
                            len = __builtin_amdgcn_readlane(x, y);
                        }
                    }
                    if (len == 0) break;
                    nb = blocks_of(len);
                }
            }
        }
        // Requests without keys
        int32_t zl = zero_len;
        for (uint32_t r = zero_r; r < R;) {
            if (nc_paged_cut(zl, max_tokens) == 0) {
                const Args z = again(args);
                for (uint32_t x = threadIdx.x; x < z->num_q_heads * D; x += THREADS)
                    z->o[r * z->o_stride + (x / D) * z->o_head_stride + x % D] = 0.f;
            }
            r += gridDim.x;
            if (r < R) zl = as_const(lens)[r];
        }
    }
};

// NEXT: heads each for themselves (MANY: where a->many says so, short ones a wave each) or neighbouring ones together, whichever
// the lengths call for; else MANY says it all.
template <int D, bool BF, bool UNI, bool MANY, bool NEXT, bool FOUR = false, bool MASS = false, int PACK = 1>
__device__ __forceinline__ void decode_body() {
    const Args a = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    using X = Decode<D, BF, UNI, MANY, false, FOUR, MASS, PACK>;
    // the waves' O, or a merge's factors, sums of rows and partial sums
    constexpr uint32_t kWaves = X::NW * 16 * X::OP, kMerge = NC_PAGED_MERGE_ROWS + 2 * 64 + 4 * X::THREADS;
    __shared__ __attribute__((aligned(16))) float s_mem[kWaves > kMerge ? kWaves : kMerge];
    __shared__ float s_ml[X::NW][16][2];
    __shared__ uint32_t s_word;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t shift = a->wave_shift, side = NEXT ? a->side : 0u;
    const int32_t *lens = a->seq_lens;
    const uint32_t max_tokens = a->max_tokens;
    const float scale = a->scale * kLog2e;
    const uint32_t R = a->num_seqs, per = (R + 63u) / 64u;  // requests of a lane
    // All of these arguments before the first load of a length: scalar loads are waited for together.
    asm volatile("" ::"s"(lens), "s"(max_tokens), "s"(R), "s"(shift), "s"(side));
    const int32_t zero_len = blockIdx.x < R ? as_const(lens)[blockIdx.x] : 1;
    uint32_t mine = 0, some = 0, len0 = 0, mine_next = 0, longest = 0;
    for (uint32_t j = 0; j < per; ++j) {
        const uint32_t r = lane * per + j;
        if (r < R) {
            len0 = nc_paged_cut(lens[r], max_tokens);
            mine += X::units_of(X::blocks_by(len0, shift));
            some += len0 != 0;
            if constexpr (NEXT) {
                mine_next += X::units_of(X::blocks_by(len0, side));
                longest = max(longest, len0);
            }
        }
    }
    auto *o = reinterpret_cast<float (*)[16][X::OP]>(s_mem);
    if constexpr (FOUR && NEXT) {  // heads each for themselves are neighbouring ones of one
        using Y = Decode<D, BF, UNI, MANY, true, FOUR, MASS, PACK>;
        const uint32_t units = (uint32_t)__builtin_amdgcn_readlane(wave_scan32(mine), 63) * a->heads.d;
        const bool next = __ballot(longest > NC_PAGED_NEXT_TOKENS) != 0 && units >= more_of(a)->next_least;
        const uint32_t by = next ? side : 0u;
        Y y{a, lane, w, lane & 15u, lane >> 4, by, Y::WK * (Y::NW >> by), w & ((1u << by) - 1u), w >> by, o, s_ml, &s_word};
        y.run(scale, next ? mine_next : mine, some, len0, zero_len);
        return;
    } else if constexpr (NEXT) {
        if (__ballot(longest > NC_PAGED_NEXT_TOKENS)) {
            using Y = Decode<D, BF, UNI, false, true>;
            Y y{a, lane, w, lane & 15u, lane >> 4, side, Y::WK * (Y::NW >> side), w & ((1u << side) - 1u), w >> side, o, s_ml, &s_word};
            y.run(scale, mine_next, some, len0, zero_len);
            return;
        }
    }
    X x{a, lane, w, lane & 15u, lane >> 4, shift, X::WK * (X::NW >> shift), w & ((1u << shift) - 1u), w >> shift, o, s_ml, &s_word};
    x.run(scale, mine, some, len0, zero_len);
}

}  // namespace

#endif
