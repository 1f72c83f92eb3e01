// paged.hip — the paged key-value cache's kernels for MI355X (gfx950, wave64): block tables and slot map
// (nc_paged_build), row append (nc_paged_append_*) and single-token attention (nc_paged_decode_*). The
// interface is described in include/notcute_paged.h. What device memory names (lengths, page ids, slots) is
// checked here before it becomes an address.

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
// Block tables, slot map and offsets: two prefix sums over the requests (new rows, pages taken). For a step of
// few tokens a request one workgroup does it all, and a request's thread writes its own slots and table entries.
// Else every slot and every new table entry finds its request by a binary search of the sums; each workgroup
// scans all requests, a workgroup's threads at a time, and does its own share of the slots and of the list.
// Latency is all there is: the lengths, the list's pages behind the sums, the stores. In a replayed graph, where an empty
// kernel takes 1.6 us: 16 requests of a token each 3.1 us, 1000 5.3, 256 prompts of 121000 rows together 5.3.
// -------------------------------------------------------------------------------------------------
extern "C" __global__ __launch_bounds__(1024) void nc_paged_build(const nc_paged_build_args a) {
    enum : uint8_t { kRefused, kGranted, kDone };
    constexpr uint32_t kFew = 8;  // rows that a request's thread writes itself
    __shared__ uint32_t s_row[1024], s_first[1024], s_held[1024], s_cached[1024];
    __shared__ uint8_t s_state[1024];
    __shared__ uint64_t s_rows[16], s_pages[16];
    __shared__ uint32_t s_taken, s_refused;

    const uint32_t tid = threadIdx.x, nt = blockDim.x, lane = tid & 63u, w = tid >> 6, nw = nt >> 6;
    const uint32_t last = gridDim.x - 1u, b = blockIdx.x;
    const bool lens = (a.parts & NC_PAGED_PART_LENS) && b == 0, pages_part = a.parts & NC_PAGED_PART_PAGES;
    const uint64_t row_lo = (uint64_t)b * a.chunk_rows;
    const uint64_t row_hi = b == last ? a.places : min((uint64_t)a.places, row_lo + a.chunk_rows);
    const uint32_t cur = (uint32_t)max(a.cursor[0], 0);
    const uint64_t list_lo = cur + (uint64_t)b * a.chunk_pages;
    const uint64_t list_hi = b == last ? a.free_len : min((uint64_t)a.free_len, list_lo + a.chunk_pages);
    const uint32_t most = a.width * a.ps.d;  // tokens of a table row
    uint64_t rows = 0, pages = cur;  // rows and list places of the requests before this pass's
    uint32_t taken = 0, refused = 0;
    if (tid == 0) s_taken = s_refused = 0;

    for (uint32_t t0 = 0; t0 < a.num_seqs; t0 += nt) {
        const uint32_t r = t0 + tid;
        uint32_t c = 0, n = 0;
        if (r < a.num_seqs) {
            c = (uint32_t)max(a.cached[r], 0);
            n = (uint32_t)max(a.fresh[r], 0);
        }
        uint32_t held = nc_paged_quot(c, a.ps);
        held += held * a.ps.d != c;
        const bool fits = (uint64_t)c + n <= most, few = gridDim.x == 1 && n <= kFew;
        int32_t *row = a.table + r * a.table_stride;
        int32_t open = -1;  // the page that the cached tokens end in, if it has places left
        if (pages_part && few && n && fits && held * a.ps.d != c) open = row[held - 1];
        uint32_t take = 0;
        if (fits) {
            const uint32_t need = nc_paged_quot(c + n, a.ps);
            take = need + (need * a.ps.d != c + n) - held;
        }
        const uint64_t rs = wave_scan64(n), ps = wave_scan64(take);
        uint64_t row0 = rows + rs - n, first = pages + ps - take, row_end = rows, page_end = pages;
        if (nw > 1) {
            if (lane == 63) {
                s_rows[w] = rs;
                s_pages[w] = ps;
            }
            __syncthreads();
            // the waves' sums, summed by every wave: lane i has those of waves 0..i
            uint64_t x = lane < nw ? s_rows[lane] : 0, y = lane < nw ? s_pages[lane] : 0;
#pragma unroll
            for (uint32_t d = 1; d < 16; d <<= 1) {
                const uint64_t u = __shfl_up(x, d, 16), v = __shfl_up(y, d, 16);
                if ((lane & 15u) >= d) {
                    x += u;
                    y += v;
                }
            }
            row0 += w ? __shfl(x, w - 1u, 64) : 0;
            first += w ? __shfl(y, w - 1u, 64) : 0;
            row_end += __shfl(x, nw - 1u, 64);
            page_end += __shfl(y, nw - 1u, 64);
        } else {
            row_end += __shfl(rs, 63, 64);
            page_end += __shfl(ps, 63, 64);
        }
        const bool ok = fits && (n == 0 || row0 + n <= a.places) && (take == 0 || first + take <= a.free_len);
        if (pages_part && few) {
            int32_t page = open;
            uint32_t in = c - (held - 1u) * a.ps.d;  // the next token's place in it; past its end without one
            uint64_t from = first;
            for (uint32_t t = 0; t < n && row0 + t < a.places; ++t) {
                if (ok && in == a.ps.d) {
                    row[held + (from - first)] = page = a.free_pages[from];
                    ++from;
                    in = 0;
                }
                a.slots[row0 + t] = ok && (uint32_t)page < a.num_pages ? (int32_t)((uint32_t)page * a.ps.d + in) : -1;
                ++in;
            }
        }
        if (pages_part && __syncthreads_or(!few)) {
            s_row[tid] = (uint32_t)min(row0, (uint64_t)a.places);
            s_first[tid] = (uint32_t)min(first, (uint64_t)a.free_len);
            s_held[tid] = held;
            s_cached[tid] = c;
            s_state[tid] = few ? kDone : ok ? kGranted : kRefused;
            __syncthreads();
            const uint64_t lo = max(min(rows, (uint64_t)a.places), row_lo), hi = min(row_end, row_hi);
            for (uint64_t i = lo + tid; i < hi; i += nt) {
                const uint32_t j = last_not_above(s_row, nt, (uint32_t)i);
                int32_t slot = -1;
                if (s_state[j] == kDone) continue;
                if (s_state[j] == kGranted) {
                    const uint32_t pos = s_cached[j] + ((uint32_t)i - s_row[j]);
                    const uint32_t at = nc_paged_quot(pos, a.ps), h = s_held[j];
                    const int32_t page = at < h ? a.table[(t0 + j) * a.table_stride + at] : a.free_pages[s_first[j] + at - h];
                    if ((uint32_t)page < a.num_pages) slot = (int32_t)((uint32_t)page * a.ps.d + (pos - at * a.ps.d));
                }
                a.slots[i] = slot;
            }
            const uint64_t plo = max(pages, list_lo), phi = min(page_end, list_hi);
            for (uint64_t e = plo + tid; e < phi; e += nt) {
                const uint32_t j = last_not_above(s_first, nt, (uint32_t)e);
                if (s_state[j] == kGranted) a.table[(t0 + j) * a.table_stride + s_held[j] + ((uint32_t)e - s_first[j])] = a.free_pages[e];
            }
        }
        if (lens && r < a.num_seqs) {
            a.seq_lens[r] = (int32_t)(ok ? c + n : c);
            a.offsets[r] = (int32_t)min(row0, (uint64_t)a.places);
            taken += ok ? take : 0;
            refused += !ok;
        }
        rows = row_end;
        pages = page_end;
        __syncthreads();  // the arrays are free again
    }
    if (pages_part)  // padding behind the last row
        for (uint64_t i = max(min(rows, (uint64_t)a.places), row_lo) + tid; i < row_hi; i += nt) a.slots[i] = -1;
    if (lens) {
        const uint32_t tk = wave_scan32(taken), rf = wave_scan32(refused);
        if (lane == 63) {
            atomicAdd(&s_taken, tk);
            atomicAdd(&s_refused, rf);
        }
        __syncthreads();
        if (tid == 0) {
            const int32_t total = (int32_t)min(rows, (uint64_t)a.places);
            a.offsets[a.num_seqs] = total;
            a.counts[0] = (int32_t)(cur + s_taken);
            a.counts[1] = total;
            a.counts[2] = (int32_t)s_taken;
            a.counts[3] = (int32_t)s_refused;
        }
    }
}

// -------------------------------------------------------------------------------------------------
// Row append: a copy, 16 bytes of K and of V per thread (more in flight per thread, or four times the rows per
// workgroup, took 2-25 % longer). What bounds it is the copy's rate. Streaming stores: 30000 rows x 8 heads x 64, off
// alignment, 26.2 -> 20.5 us (6.0 TB/s of rows read and written), 2048 x 8 x 128 4.1 -> 3.5 us; but where a head's
// row is 32 bytes and stands alone (page size 1) 8.6 -> 10.7 us, so not for head_dim 16. VEC: the rows are
// 16-byte aligned.
// -------------------------------------------------------------------------------------------------
namespace {

template <bool VEC>
__device__ __forceinline__ u32x4 load8(const uint16_t *p) {
    u32x4 r;
    if constexpr (VEC)
        r = *reinterpret_cast<const u32x4 *>(p);
    else
        __builtin_memcpy(&r, p, 16);  // one load: global memory takes them at any alignment
    return r;
}

template <bool VEC, bool STREAM>
__device__ __forceinline__ void append_body(const nc_paged_append_args &a) {
    const uint64_t row0 = (uint64_t)blockIdx.x * a.wg_rows;
    const uint32_t rows = (uint32_t)min((uint64_t)a.wg_rows, a.num_rows - row0), total = rows * a.chunks.d;
    for (uint32_t u = threadIdx.x; u < total; u += blockDim.x) {
        const uint32_t i = nc_paged_quot(u, a.chunks), c = u - i * a.chunks.d;
        const uint32_t h = c >> a.chunk_shift, x = c & ((1u << a.chunk_shift) - 1u);
        const uint32_t slot = (uint32_t)a.slots[row0 + i];
        if (slot >= a.num_slots) continue;
        const uint32_t page = nc_paged_quot(slot, a.ps), t = slot - page * a.ps.d;
        const uint64_t src = (row0 + i) * a.row_stride + h * a.row_head_stride + 8 * x;
        const uint64_t dst = page * a.page_stride + h * a.head_stride + t * a.token_stride + 8 * x;
        const u32x4 kv = load8<VEC>(a.k_rows + src), vv = load8<VEC>(a.v_rows + src);
        u32x4 *kd = reinterpret_cast<u32x4 *>(a.k + dst), *vd = reinterpret_cast<u32x4 *>(a.v + dst);
        if constexpr (STREAM) {
            __builtin_nontemporal_store(kv, kd);
            __builtin_nontemporal_store(vv, vd);
        } else {
            *kd = kv;
            *vd = vv;
        }
    }
}

}  // namespace

#define NC_APPEND(T, VEC, STREAM)                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void nc_paged_append_rows##T(const nc_paged_append_args a) {          \
        append_body<VEC, STREAM>(a);                                                                                  \
    }
NC_APPEND(, true, true)
NC_APPEND(_unaligned, false, true)
NC_APPEND(_d16, true, false)
NC_APPEND(_d16_unaligned, false, false)

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
template <bool BF>
__device__ __forceinline__ uint32_t take_pair(float &x, float &y) {
    if constexpr (BF) {
        const bf16x2 h = {(__bf16)x, (__bf16)y};
        const uint32_t u = __builtin_bit_cast(uint32_t, h);
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

template <int D, bool BF, bool UNI, bool MANY, bool NEXT>
struct Decode {
    static constexpr int KT = D <= 32 ? 2 : 1;  // 32-key tiles of a wave's step
    static constexpr int NT = 2 * KT;           // 16-key tiles
    static constexpr uint32_t WK = 32 * KT;     // keys of a wave's step: nc_paged_step_keys(D)
    static constexpr int E = D / 16;            // dims of a lane in V and O
    static constexpr int KK = D < 32 ? 1 : D / 32;  // products of a score
    static constexpr int KE = D == 16 ? 4 : 8;  // dims of a lane in one product
    // Whether a step's loads are under way before the one before it is computed. It costs registers, and pays where a step's
    // loads are wide and heads end at different times: 64 ragged requests over 4 heads of 64 31.6 -> 28.7 us, 32 of 2048 over 8
    // of 64 28.0 -> 27.6 (but one of 120001 over 8 of 64, token-major, 53 -> 56). Heads of 16 or 32 are better off with more
    // workgroups instead (33 requests of up to 2047, 16 heads of 32, 11.9 -> 11.1 us on pages of 16, and 14.4 -> 11.4 of 7), and
    // with heads of 128 on odd pages both the addresses and two steps do not fit (1 % slower).
    static constexpr bool AHEAD = D == 64 || (D == 128 && UNI);
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
    using VReg = typename std::conditional<E == 8, u32x4, typename std::conditional<E == 4, u32x2, uint32_t>::type>::type;

    // K and V of a wave's step, on their way or there, and which keys count: the first seen[t] of a tile, or
    // (pages of any size) those whose bits are set in it.
    struct Step {
        KReg k[NT][KK];
        VReg v[NT][4];
        uint32_t seen[NT];
    };
    struct Pages {
        uint32_t e[NT];
    };
    // One request's table row and one key head of the pools. Off: a page fits 32 bits where a tile lies in one.
    using Off = typename std::conditional<UNI, uint32_t, uint64_t>::type;
    struct Cache {
        const int32_t *table;
        const uint16_t *k, *v;
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
    u32x4 qv[KK];
    floatx4 acc[E];
    float m, l;

    // Blocks of WK * (NW >> shift) keys.
    static __device__ __forceinline__ uint32_t blocks_by(uint32_t len, uint32_t shift) {
        return (len + (WK * NW >> shift) - 1u) >> (__builtin_ctz(WK * NW) - shift);
    }
    __device__ __forceinline__ uint32_t blocks_of(uint32_t len) const { return blocks_by(len, wave_shift); }
    // Query heads of a piece.
    __device__ __forceinline__ uint32_t piece_rows(Args a) const { return NEXT ? a->group << wave_shift : a->rows; }
    static __device__ __forceinline__ uint32_t units_of(uint32_t nb) { return nb ? nb + nc_paged_head_units(D) : 0u; }

    // Q of a block's query heads as the B operand: lane (c, g) holds query c of the wave's 16, dims KE*g.. of 32.
    __device__ __forceinline__ void load_q(uint32_t r, uint32_t head0, uint32_t rows) {
        const Args a = again(args);
        const uint32_t row = NEXT ? qt * a->group + min(c, a->group - 1u) : min(16u * qt + c, rows - 1u);
        const uint16_t *p = a->q + r * a->q_stride + (head0 + row) * a->q_head_stride;
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

    // A raw buffer of `bytes` bytes.
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(const uint16_t *p, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(p), 0, (int)bytes, 0x00020000);
    }

    static __device__ __forceinline__ uint32_t word(const VReg &v, int i) {
        if constexpr (E > 2)
            return v[i];
        else
            return v;
    }

    __device__ __forceinline__ void compute(Step &st) {
        bool full = true;
#pragma unroll
        for (int t = 0; t < NT; ++t) full = full && st.seen[t] == (UNI ? 16u : 0xffffu);
        float s[NT][4];
        float top = neg_inf();
        floatx4 dot[NT];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const floatx4 x = kk ? dot[t] : floatx4{0.f, 0.f, 0.f, 0.f};
                if constexpr (D == 16)
                    dot[t] = mfma_k16<BF>(st.k[t][kk], u32x2{qv[kk][0], qv[kk][1]}, x);
                else
                    dot[t] = mfma_k32<BF>(st.k[t][kk], qv[kk], x);
            }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = dot[t][i] * sc;
        if (!full) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = UNI ? 4 * g + i < st.seen[t] : st.seen[t] >> (4 * g + i) & 1u;
                    s[t][i] = in ? s[t][i] : neg_inf();
                    if constexpr (!UNI) {  // 0 * NaN would be NaN
                        if constexpr (E > 2) {
#pragma unroll
                            for (int j = 0; j < E / 2; ++j) st.v[t][i][j] = in ? st.v[t][i][j] : 0u;
                        } else {
                            st.v[t][i] = in ? st.v[t][i] : 0u;
                        }
                    }
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
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
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - ref) * UNIT;
                l += s[t][i];
            }
        u32x4 p[KT][PARTS];
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < PARTS; ++n)
                    p[u][n][j] = take_pair<BF>(s[2 * u + j / 2][2 * (j % 2)], s[2 * u + j / 2][2 * (j % 2) + 1]);
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
                        const uint32_t lo = word(st.v[2 * u + j / 2][2 * (j % 2)], (i0 + i) / 2);
                        const uint32_t hi = word(st.v[2 * u + j / 2][2 * (j % 2) + 1], (i0 + i) / 2);
                        x[i][j] = __builtin_amdgcn_perm(hi, lo, i % 2 ? 0x07060302u : 0x05040100u);
                    }
#pragma unroll
                for (int n = 0; n < PARTS; ++n)
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        floatx4 &sum = n ? low[i] : acc[i0 + i];
                        sum = mfma_k32<BF>(x[i], p[u][n], sum);
                    }
            }
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
        cache.k = a->k + kvh * a->head_stride;
        cache.v = a->v + kvh * a->head_stride;
        cache.page_stride = a->page_stride;
        cache.token_stride = a->token_stride;
        cache.num_pages = a->num_pages;
        cache.ps.d = a->ps.d;
        cache.ps.magic = a->ps.magic;
        cache.ps.shift = a->ps.shift;
        Step x, y;
        Pages pages = load_pages(cache, k0, len);
        issue(x, cache, pages, k0, end);
        if constexpr (!AHEAD) {
            while (true) {
                pages = load_pages(cache, k0 + by, len);
                compute(x);
                if ((k0 += by) >= end) return;
                issue(x, cache, pages, k0, end);
            }
        }
        if (k0 + by >= end) {
            compute(x);
            return;
        }
        pages = load_pages(cache, k0 + by, len);
        while (true) {
            issue(y, cache, pages, k0 + by, end);
            pages = load_pages(cache, k0 + 2 * by, len);
            compute(x);
            if (k0 + by >= end) break;
            issue(x, cache, pages, k0 + 2 * by, end);
            pages = load_pages(cache, k0 + 3 * by, len);
            compute(y);
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
            store_o(o, q, x, out, sum);
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
                    store_o(o, q, x, out, s_tot[2 * q + 1]);
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

    __device__ __forceinline__ void store_o(float *o, uint32_t q, uint32_t x, floatx4 v, float sum) {
        const float inv = __builtin_amdgcn_rcpf(sum);  // to an ulp
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

    // O of a head that the wave had to itself: lane (c, g) has dims 4gE..4gE+4E-1 of query c.
    __device__ __forceinline__ void finish_wave(uint32_t r, uint32_t head0, uint32_t rows) {
        const Args a = again(args);
        const float sum = quad_sum(l);
        if (c >= rows) return;
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
                store_o(o, q, x, out, lsum);
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
        kat = 2u * (c * (uint32_t)a->token_stride + KE * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) vat[i] = 2u * ((4 * g + i) * (uint32_t)a->token_stride + E * c);
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
                const uint32_t b_lo = seg + nc_paged_head_units(D);  // unit of block 0
                uint32_t b0 = u0 > b_lo ? u0 - b_lo : 0u, b1 = u1 > b_lo ? min(nb, u1 - b_lo) : 0u;
                if (short_head) {  // all of it is the workgroup's that has its first unit
                    b0 = 0;
                    b1 = seg >= u0 ? nb : 0u;
                }
                // Short heads of a request in a row, whose first units are here: a wave each if that takes no more steps than
                // there are heads.
                uint32_t n = 1;
                if constexpr (MANY) {
                    if (nb == 1 && seg >= u0 && a->many) {
                        n = min(min(heads - head, NW), (u1 - seg + units_of(1) - 1u) / units_of(1));
                        if (len > n * WK) n = 1;
                    }
                }
                const bool alone = MANY && n > 1;
                if (alone ? w < n : b0 < b1) {
                    uint32_t kvh = alone ? head + w : head, part = 0;
                    if constexpr (NEXT) {
                        kvh = (head << wave_shift) + qt;
                    } else if (a->head_parts > 1) {
                        kvh = head / a->head_parts;
                        part = head - kvh * a->head_parts;
                    }
                    const uint32_t rows = NEXT ? piece_rows(a) : min(64u, a->group - 64u * part);
                    const uint32_t head0 = NEXT ? head * rows : kvh * a->group + 64u * part;
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
template <int D, bool BF, bool UNI, bool MANY, bool NEXT>
__device__ __forceinline__ void decode_body() {
    const Args a = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    using X = Decode<D, BF, UNI, MANY, false>;
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
    if constexpr (NEXT) {
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

// `_odd`: pages of any size; the others take sizes that are multiples of 16. `_many`: a wave may take a head for itself.
// `_next`: the waves take neighbouring heads of long requests.
#define NC_DECODE_KERNEL(NAME, D, BF, UNI, MANY, NEXT)                                                    \
    extern "C" __global__ __launch_bounds__(64 * NC_PAGED_WAVES, 2) void NAME(const nc_paged_decode_args) { \
        decode_body<D, BF, UNI, MANY, NEXT>();                                                            \
    }
#define NC_DECODE(D, T, BF)                                                       \
    NC_DECODE_KERNEL(nc_paged_decode_d##D##T, D, BF, true, false, false)           \
    NC_DECODE_KERNEL(nc_paged_decode_d##D##_odd##T, D, BF, false, false, false)    \
    NC_DECODE_KERNEL(nc_paged_decode_d##D##_many##T, D, BF, true, true, false)     \
    NC_DECODE_KERNEL(nc_paged_decode_d##D##_many_odd##T, D, BF, false, true, false) \
    NC_DECODE_KERNEL(nc_paged_decode_d##D##_next##T, D, BF, true, true, true)     \
    NC_DECODE_KERNEL(nc_paged_decode_d##D##_next_odd##T, D, BF, false, true, true)
NC_DECODE(16, , false)
NC_DECODE(32, , false)
NC_DECODE(64, , false)
NC_DECODE(128, , false)
NC_DECODE(16, _bf16, true)
NC_DECODE(32, _bf16, true)
NC_DECODE(64, _bf16, true)
NC_DECODE(128, _bf16, true)
