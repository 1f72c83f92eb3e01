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

__device__ __forceinline__ uint64_t wave_scan(uint64_t x, uint32_t lane) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    return x;
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
// Block tables, slot map and offsets. Two prefix sums over the requests (new rows, pages taken), then
// every slot and every new table entry finds its request by a binary search of them. Each workgroup
// scans all requests, a workgroup's threads at a time, and does its own share of the slots and of the list:
// for a step of one token a request the scan is all there is, and one workgroup does everything.
// -------------------------------------------------------------------------------------------------
extern "C" __global__ __launch_bounds__(1024) void nc_paged_build(const nc_paged_build_args a) {
    __shared__ uint32_t s_row[1024], s_first[1024], s_held[1024], s_cached[1024];
    __shared__ uint8_t s_ok[1024];
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
    uint64_t rows = 0, pages = cur;  // rows and list places of the requests before this round's
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
        const bool fits = (uint64_t)c + n <= most;
        uint32_t take = 0;
        if (fits) {
            const uint32_t need = nc_paged_quot(c + n, a.ps);
            take = need + (need * a.ps.d != c + n) - held;
        }
        const uint64_t rs = wave_scan(n, lane), ps = wave_scan(take, lane);
        if (lane == 63) {
            s_rows[w] = rs;
            s_pages[w] = ps;
        }
        __syncthreads();
        uint64_t row0 = rows + rs - n, first = pages + ps - take, row_end = rows, page_end = pages;
        for (uint32_t i = 0; i < nw; ++i) {
            const uint64_t x = s_rows[i], y = s_pages[i];
            if (i < w) {
                row0 += x;
                first += y;
            }
            row_end += x;
            page_end += y;
        }
        const bool ok = fits && (n == 0 || row0 + n <= a.places) && (take == 0 || first + take <= a.free_len);
        if (pages_part) {
            s_row[tid] = (uint32_t)min(row0, (uint64_t)a.places);
            s_first[tid] = (uint32_t)min(first, (uint64_t)a.free_len);
            s_held[tid] = held;
            s_cached[tid] = c;
            s_ok[tid] = ok;
            __syncthreads();
            const uint64_t lo = max(min(rows, (uint64_t)a.places), row_lo), hi = min(row_end, row_hi);
            for (uint64_t i = lo + tid; i < hi; i += nt) {
                const uint32_t j = last_not_above(s_row, nt, (uint32_t)i);
                int32_t slot = -1;
                if (s_ok[j]) {
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
                if (s_ok[j]) a.table[(t0 + j) * a.table_stride + s_held[j] + ((uint32_t)e - s_first[j])] = a.free_pages[e];
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
        const uint32_t tk = (uint32_t)wave_scan(taken, lane), rf = (uint32_t)wave_scan(refused, lane);
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
// Row append: a copy, 16 bytes of K and of V per thread and step. VEC: the rows are 16-byte aligned.
// -------------------------------------------------------------------------------------------------
namespace {

template <bool VEC>
__device__ __forceinline__ u32x4 load8(const uint16_t *p) {
    if constexpr (VEC) {
        return *reinterpret_cast<const u32x4 *>(p);
    } else {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = uint32_t(p[2 * i]) | (uint32_t(p[2 * i + 1]) << 16);
        return r;
    }
}

template <bool VEC>
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
        *reinterpret_cast<u32x4 *>(a.k + dst) = kv;
        *reinterpret_cast<u32x4 *>(a.v + dst) = vv;
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void nc_paged_append_rows(const nc_paged_append_args a) { append_body<true>(a); }
extern "C" __global__ __launch_bounds__(256) void nc_paged_append_rows_unaligned(const nc_paged_append_args a) {
    append_body<false>(a);
}

// -------------------------------------------------------------------------------------------------
// Single-token attention. Up to 16 query heads of one key head are the 16 columns of the matrix products, so
// K and V are read once for all of them; with up to 64, two or four waves of a workgroup take the same keys at
// the same time, and all but one find them in the caches. The work is cut into blocks, counted over all requests
// and heads, and every workgroup takes a run of equally many, whatever the lengths: it finds its first by a
// prefix sum over the requests' lengths. A run that begins or ends inside a request's keys leaves a piece
// (max, sum, O); the last of a request's workgroups to arrive joins them in order.
//
// One wave takes KT x 32 keys of a block at a time. Scores: S = K Q^T with K rows straight from memory as the
// A operand (lane l: key l%16, dims 8(l/16)..+7 of 32), so lane l holds the scores of query l%16 and keys
// 4(l/16)+r of each 16. These registers are the B operand of O^T += V^T P^T as they stand, if V's k index runs
// the same way: the lane loads D/16 dims of the eight keys 16t + 4(l/16) + r and turns them in registers.
// Nothing but the final join of the four waves goes through LDS. K and V are read once and the rest is small, so
// the read rate bounds it; the matrix cores have time for weights in two (f16) or three (bf16) parts, whose
// sum is the f32 weight to 2^-21 or better: rounding them to one 16-bit number would cost 2^-12 or 2^-9.
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

// Two f32 rounded to nearest as a pair of 16-bit numbers; x and y become what that leaves.
template <bool BF>
__device__ __forceinline__ uint32_t take_pair(float &x, float &y) {
    if constexpr (BF) {
        const bf16x2 h = {(__bf16)x, (__bf16)y};
        x -= (float)h[0];
        y -= (float)h[1];
        return __builtin_bit_cast(uint32_t, h);
    } else {
        const half2v h = {(_Float16)x, (_Float16)y};
        x -= (float)h[0];
        y -= (float)h[1];
        return __builtin_bit_cast(uint32_t, h);
    }
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

__device__ __forceinline__ uint32_t wave_scan32(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
    return x;
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

__device__ __forceinline__ float finite_or_0(float m) { return m == neg_inf() ? 0.f : m; }

// Which keys a workgroup is at: request r of length len, whose blocks begin behind `pre` blocks of the
// requests before it.
struct Place {
    uint32_t r, len, pre;
};

template <int D, bool BF, bool UNI>
struct Decode {
    static constexpr int KT = D == 16 ? 4 : D == 32 ? 2 : 1;  // 32-key tiles of a wave's step
    static constexpr int NT = 2 * KT;                        // 16-key tiles
    static constexpr uint32_t WK = 32 * KT;                  // keys of a wave's step: nc_paged_step_keys(D)
    static constexpr int E = D / 16;                         // dims of a lane in V and O
    static constexpr int KK = D < 32 ? 1 : D / 32;           // products of a score
    static constexpr int OP = D + 4;                         // pitch of a row of partial O in LDS
    // Weights are 2^(SHIFT + score - max): in f16 the low part of a small weight stays a normal number, in bf16
    // a sum of a million V at the type's largest value stays finite.
    static constexpr float SHIFT = BF ? -16.f : 12.f;
    using KReg = typename std::conditional<D == 16, u32x2, u32x4>::type;

    const nc_paged_decode_args &a;
    const uint32_t lane, w, c, g;
    const uint32_t bk;  // keys of a block
    float (*s_o)[16][OP];   // [4]
    float (*s_ml)[16][2];   // [4]
    uint32_t *s_word;

    u32x4 qv[KK];
    floatx4 acc[E];
    float m, l;

    // bk = WK * 2^(2 - wave_shift)
    __device__ __forceinline__ uint32_t blocks_of(uint32_t len) const {
        return (len + bk - 1) >> (__builtin_ctz(WK) + 2 - a.wave_shift);
    }

    // Q of the block's query heads as the B operand: lane (c, g) holds query c, dims 8g.. (4g.. for D = 16).
    __device__ __forceinline__ void load_q(uint32_t r, uint32_t head0, uint32_t row, uint32_t rows) {
        const uint16_t *p = a.q + r * a.q_stride + (head0 + min(row + c, rows - 1u)) * a.q_head_stride;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            constexpr int N = D == 16 ? 4 : 8;
            const uint16_t *x = p + 32 * kk + N * g;
            u32x4 t = {0u, 0u, 0u, 0u};
            if (a.q_vec) {
                if constexpr (D == 16) {
                    const u32x2 y = *reinterpret_cast<const u32x2 *>(x);
                    t[0] = y[0];
                    t[1] = y[1];
                } else {
                    t = *reinterpret_cast<const u32x4 *>(x);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) t[i] = uint32_t(x[2 * i]) | uint32_t(x[2 * i + 1]) << 16;
            }
            qv[kk] = t;
        }
    }

    // Table entries of a step's 16-key tiles: uniform where a tile lies in one page, else one per lane (key c
    // of the tile). Past the request's end the last key's entry.
    __device__ __forceinline__ void load_pages(uint32_t (&e)[NT], uint64_t row, uint32_t k0, uint32_t len) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (UNI)
                e[t] = (uint32_t)as_const(a.table)[row + nc_paged_quot(min(k0 + 16 * t, len - 1u), a.ps)];
            else
                e[t] = (uint32_t)a.table[row + nc_paged_quot(min(k0 + 16 * t + c, len - 1u), a.ps)];
        }
    }

    // One step: the keys k0..k0+WK-1 of a request of length len, k0 < len, on the pages e.
    __device__ __forceinline__ void step(const uint32_t (&e)[NT], uint32_t k0, uint32_t len, uint32_t kvh) {
        KReg kr[NT][KK];
        u32x4 vr[NT][4];  // E dims in the first E/2 dwords (D = 16: half of one)
        uint32_t seen[NT];  // bit i: key i of the tile counts
        const uint16_t *kh = a.k + kvh * a.head_stride, *vh = a.v + kvh * a.head_stride;
        const uint16_t *vb[NT][4];
        auto load_k = [&](int t, const uint16_t *p) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) kr[t][kk] = *reinterpret_cast<const KReg *>(p + 32 * kk);
        };
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t k1 = k0 + 16 * t;
            if constexpr (UNI) {
                // A tile without keys, or on a page outside the pool, reads the pool's page 0 and counts for nothing.
                const bool in = k1 < len && e[t] < a.num_pages;
                seen[t] = in ? (k1 + 16 <= len ? 0xffffu : (1u << (len - k1)) - 1u) : 0u;
                const uint32_t ka = min(k1, (len - 1u) & ~15u);  // below 2^31
                const uint64_t at = (in ? e[t] : 0u) * a.page_stride + (ka - nc_paged_quot(ka, a.ps) * a.ps.d) * a.token_stride;
                const uint32_t ts = (uint32_t)a.token_stride;
                load_k(t, kh + at + (c * ts + (D == 16 ? 4 : 8) * g));
#pragma unroll
                for (int i = 0; i < 4; ++i) vb[t][i] = vh + at + ((4 * g + i) * ts + E * c);
            } else {
                const uint32_t key = min(k1 + c, len - 1u);
                const bool in = k1 + c < len && e[t] < a.num_pages;
                seen[t] = (uint32_t)__ballot(in) & 0xffffu;
                const uint64_t at = (in ? e[t] : 0u) * a.page_stride + (key - nc_paged_quot(key, a.ps) * a.ps.d) * a.token_stride;
                load_k(t, kh + at + (D == 16 ? 4 : 8) * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int from = 4 * (int)g + i;
                    const uint32_t lo = __shfl((uint32_t)at, from, 64), hi = __shfl((uint32_t)(at >> 32), from, 64);
                    vb[t][i] = vh + ((uint64_t)hi << 32 | lo) + E * c;
                }
            }
        }
        bool full = true;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            full = full && seen[t] == 0xffffu;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (E == 8) {
                    vr[t][i] = *reinterpret_cast<const u32x4 *>(vb[t][i]);
                } else if constexpr (E == 4) {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(vb[t][i]);
                    vr[t][i][0] = x[0];
                    vr[t][i][1] = x[1];
                } else if constexpr (E == 2) {
                    vr[t][i][0] = *reinterpret_cast<const uint32_t *>(vb[t][i]);
                } else {
                    vr[t][i][0] = *vb[t][i];
                }
            }
        }

        float s[NT][4];
        const float sc = a.scale * kLog2e;
        float top = neg_inf();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                if constexpr (D == 16)
                    x = mfma_k16<BF>(kr[t][kk], u32x2{qv[kk][0], qv[kk][1]}, x);
                else
                    x = mfma_k32<BF>(kr[t][kk], qv[kk], x);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = x[i] * sc;
        }
        if (!full) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = seen[t] >> (4 * g + i) & 1u;
                    s[t][i] = in ? s[t][i] : neg_inf();
#pragma unroll
                    for (int j = 0; j < (E + 1) / 2; ++j) vr[t][i][j] = in ? vr[t][i][j] : 0u;  // 0 * NaN would be NaN
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
        top = fmaxf(m, quad_max(top));
        const float ref = finite_or_0(top) - SHIFT;
        if (!__all(top == m)) {
            const float f = __builtin_amdgcn_exp2f(m - finite_or_0(top));
            l *= f;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] *= f;
            m = top;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - ref);
                l += s[t][i];
            }
        constexpr int PARTS = BF ? 3 : 2;
#pragma unroll
        for (int u = 0; u < KT; ++u) {
            u32x4 p[PARTS];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < PARTS; ++n) p[n][j] = take_pair<BF>(s[2 * u + j / 2][2 * (j % 2)], s[2 * u + j / 2][2 * (j % 2) + 1]);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                u32x4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t lo = vr[2 * u + j / 2][2 * (j % 2)][i / 2], hi = vr[2 * u + j / 2][2 * (j % 2) + 1][i / 2];
                    x[j] = __builtin_amdgcn_perm(hi, lo, i % 2 ? 0x07060302u : 0x05040100u);
                }
#pragma unroll
                for (int n = 0; n < PARTS; ++n) acc[i] = mfma_k32<BF>(x, p[n], acc[i]);
            }
        }
    }

    // The pieces of workgroups first..last of one request and head: added in an order that does not depend on who
    // came last, and written to O. Four columns of a row are a thread's; where that leaves threads over, groups of
    // them take every so many-th piece and are added up through LDS. PF pieces are on their way at a time.
    template <int PF>
    __device__ __forceinline__ void join_pieces(uint32_t first, uint32_t last, uint32_t rows, float *o) {
        const uint32_t items = rows * (D / 4), groups = items > 128 ? 1u : 256u / items;
        floatx4 *s_sum = reinterpret_cast<floatx4 *>(&s_o[0][0][0]);  // one per thread, and behind them (max, sum)
        float *s_stat = reinterpret_cast<float *>(s_sum + 256);
        for (uint32_t i0 = 0; i0 < items; i0 += 256) {
            const uint32_t grp = groups == 1 ? 0u : threadIdx.x / items, it = groups == 1 ? i0 + threadIdx.x : threadIdx.x - grp * items;
            const bool mine = it < items && grp < groups;
            const uint32_t q = it / (D / 4), x = 4 * (it % (D / 4));
            float top = neg_inf(), sum = 0.f;
            floatx4 out = {0.f, 0.f, 0.f, 0.f};
            if (mine) {
                for (uint32_t i = first + grp; i <= last; i += PF * groups) {
                    float pm[PF], pl[PF];
                    floatx4 po[PF];
#pragma unroll
                    for (int n = 0; n < PF; ++n) {
                        const uint32_t j = min(i + n * groups, last);
                        const uint64_t at = ((uint64_t)j * 2 + (j == first)) * a.rows + q;
                        float p0, p1, p2, p3;
                        get2(a.part_ml + 2 * at, pm[n], pl[n]);
                        get2(a.part_o + at * D + x, p0, p1);
                        get2(a.part_o + at * D + x + 2, p2, p3);
                        po[n] = floatx4{p0, p1, p2, p3};
                    }
                    float t = top;
#pragma unroll
                    for (int n = 0; n < PF; ++n) {
                        if (i + n * groups > last) pm[n] = neg_inf();
                        t = fmaxf(t, pm[n]);
                    }
                    const float ref = finite_or_0(t), f = __builtin_amdgcn_exp2f(top - ref);
                    sum *= f;
                    out *= f;
#pragma unroll
                    for (int n = 0; n < PF; ++n) {
                        if (i + n * groups <= last) {
                            const float h = __builtin_amdgcn_exp2f(pm[n] - ref);
                            sum += pl[n] * h;
                            out += po[n] * h;
                        }
                    }
                    top = t;
                }
            }
            if (groups > 1) {
                s_sum[threadIdx.x] = out;
                s_stat[2 * threadIdx.x] = top;
                s_stat[2 * threadIdx.x + 1] = sum;
                __syncthreads();
                if (mine && grp == 0) {
                    float t = top;
                    for (uint32_t n = 1; n < groups; ++n) t = fmaxf(t, s_stat[2 * (threadIdx.x + n * items)]);
                    const float ref = finite_or_0(t), f = __builtin_amdgcn_exp2f(top - ref);
                    sum *= f;
                    out *= f;
                    for (uint32_t n = 1; n < groups; ++n) {
                        const uint32_t y = threadIdx.x + n * items;
                        const float h = __builtin_amdgcn_exp2f(s_stat[2 * y] - ref);
                        sum += s_stat[2 * y + 1] * h;
                        out += s_sum[y] * h;
                    }
                }
            }
            if (mine && grp == 0) store_o(o, q, x, out, sum);
        }
    }

    __device__ __forceinline__ void store_o(float *o, uint32_t q, uint32_t x, floatx4 v, float sum) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = sum == 0.f ? 0.f : v[i] / sum;
        float *p = o + q * a.o_head_stride + x;
        if (a.o_vec) {
            *reinterpret_cast<floatx4 *>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = v[i];
        }
    }

    // The four waves' (m, l, O) of one run of blocks: to O if the run is all of the request's, else to this
    // workgroup's (i's) piece, and the last of workgroups first..last to arrive joins them.
    __device__ __forceinline__ void finish(uint32_t rows, float *o, bool whole, uint32_t i, uint32_t first, uint32_t last) {
        const float sum = quad_sum(l);
        if (g == 0) {
            s_ml[w][c][0] = m;
            s_ml[w][c][1] = sum;
        }
        if (16 * (w & ((1u << a.wave_shift) - 1u)) + c < rows) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < E; ++j) s_o[w][c][(4 * g + r) * E + j] = acc[j][r];
        }
        __syncthreads();
        const uint32_t items = rows * (D / 4);
        for (uint32_t it = threadIdx.x; it < items; it += 256) {
            const uint32_t q = it / (D / 4), x = 4 * (it % (D / 4));
            const uint32_t q16 = q & 15u, by = 1u << a.wave_shift;  // waves q / 16, + by, ... hold query q
            float top = neg_inf(), lsum = 0.f;
            for (uint32_t n = q >> 4; n < 4; n += by) top = fmaxf(top, s_ml[n][q16][0]);
            floatx4 out = {0.f, 0.f, 0.f, 0.f};
            for (uint32_t n = q >> 4; n < 4; n += by) {
                const float f = __builtin_amdgcn_exp2f(s_ml[n][q16][0] - finite_or_0(top));
                lsum += f * s_ml[n][q16][1];
                out += f * *reinterpret_cast<const floatx4 *>(&s_o[n][q16][x]);
            }
            if (whole) {
                store_o(o, q, x, out, lsum);
            } else {
                const uint64_t at = ((uint64_t)i * 2 + (i == first)) * a.rows + q;
                put2(a.part_o + at * D + x, out[0], out[1]);
                put2(a.part_o + at * D + x + 2, out[2], out[3]);
                if (x == 0) put2(a.part_ml + 2 * at, top, lsum);
            }
        }
        if (!whole) {
            // Every thread's stores have arrived before the count says so, and the partials are read only after the
            // count showed the last of them.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0)
                *s_word = __hip_atomic_fetch_add(a.counters + first, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (*s_word == last - first) {
                const uint32_t pieces = (last - first + 1) * min(rows * (D / 4), 256u);  // a thread's, times 256
                if (pieces <= 2 * 256)
                    join_pieces<2>(first, last, rows, o);
                else if (pieces <= 4 * 256)
                    join_pieces<4>(first, last, rows, o);
                else
                    join_pieces<8>(first, last, rows, o);
                if (threadIdx.x == 0) __hip_atomic_store(a.counters + first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        __syncthreads();  // LDS is free again
    }

    __device__ __forceinline__ void run() {
        const uint32_t R = a.num_seqs, per = (R + 63u) / 64u;  // requests of a lane
        const uint32_t heads = a.num_kv_heads * a.head_parts;
        const uint32_t qt = w & ((1u << a.wave_shift) - 1u), kw = w >> a.wave_shift;  // query heads' and keys' part
        const uint32_t zero_r = blockIdx.x;
        const int32_t zero_len = zero_r < R ? as_const(a.seq_lens)[zero_r] : 1;
        uint32_t mine = 0, len0 = 0;
        for (uint32_t j = 0; j < per; ++j) {
            const uint32_t r = lane * per + j;
            if (r < R) {
                len0 = nc_paged_cut(a.seq_lens[r], a.max_tokens);
                mine += blocks_of(len0);
            }
        }
        const uint32_t incl = wave_scan32(mine);
        const uint32_t blocks = __builtin_amdgcn_readlane(incl, 63) * heads, i = blockIdx.x;
        const uint32_t each = nc_paged_each(blocks, gridDim.x);
        uint32_t b = i * each;
        if (b < blocks) {
            const uint32_t end = min(b + each, blocks);
            Place at;
            {
                const uint32_t t = b / heads;  // the same request's block if it had one head
                const uint32_t from = __builtin_ctzll(__ballot(incl - mine <= t && t < incl));
                at.pre = __builtin_amdgcn_readlane(incl - mine, from);
                at.r = from * per;
                at.len = __builtin_amdgcn_readlane(len0, from);
                if (per > 1) {
                    const uint32_t r0 = at.r, most = min(per, R - r0);
                    for (uint32_t x = 0; x < most; x += 64) {
                        const uint32_t len = x + lane < most ? nc_paged_cut(a.seq_lens[r0 + x + lane], a.max_tokens) : 0u;
                        const uint32_t nb = blocks_of(len), sc = wave_scan32(nb);
                        const uint64_t hit = __ballot(t < at.pre + sc);
                        if (hit) {
                            const uint32_t y = __builtin_ctzll(hit);
                            at.r = r0 + x + y;
                            at.len = __builtin_amdgcn_readlane(len, y);
                            at.pre += __builtin_amdgcn_readlane(sc - nb, y);
                            break;
                        }
                        at.pre += __builtin_amdgcn_readlane(sc, 63);
                    }
                }
            }
            uint32_t nb = blocks_of(at.len);
            uint32_t head = (b - at.pre * heads) / nb, b0 = b - at.pre * heads - head * nb;
            while (true) {
                const uint32_t b1 = min(nb, b0 + (end - b));
                const uint32_t kvh = head / a.head_parts, part = head - kvh * a.head_parts;
                const uint32_t rows = min(64u, a.group - 64u * part), head0 = kvh * a.group + 64u * part;
                load_q(at.r, head0, 16u * qt, rows);
                m = neg_inf();
                l = 0.f;
#pragma unroll
                for (int x = 0; x < E; ++x) acc[x] = floatx4{0.f, 0.f, 0.f, 0.f};
                uint32_t k0 = b0 * bk + kw * WK;
                const uint32_t k1 = min(b1 * bk, at.len);
                const uint64_t row = at.r * a.table_stride;
                if (k0 < k1) {
                    uint32_t e[NT];
                    load_pages(e, row, k0, at.len);
                    while (true) {
                        uint32_t next[NT];
                        load_pages(next, row, k0 + bk, at.len);
                        step(e, k0, at.len, kvh);
                        k0 += bk;
                        if (k0 >= k1) break;
#pragma unroll
                        for (int t = 0; t < NT; ++t) e[t] = next[t];
                    }
                }
                const uint32_t seg = at.pre * heads + head * nb;  // the request's and head's first block
                const bool whole = b0 == 0 && b1 == nb;
                finish(rows, a.o + at.r * a.o_stride + head0 * a.o_head_stride, whole, i, seg / each, (seg + nb - 1) / each);
                b += b1 - b0;
                if (b >= end) break;
                b0 = 0;
                if (++head == heads) {
                    head = 0;
                    at.pre += nb;
                    do at.len = ++at.r < R ? nc_paged_cut(as_const(a.seq_lens)[at.r], a.max_tokens) : 1u;
                    while (at.len == 0);  // the share has blocks left, so there is one
                    if (at.r >= R) break;
                    nb = blocks_of(at.len);
                }
            }
        }
        // Requests without keys
        int32_t zl = zero_len;
        for (uint32_t r = zero_r; r < R;) {
            if (nc_paged_cut(zl, a.max_tokens) == 0)
                for (uint32_t x = threadIdx.x; x < a.num_q_heads * D; x += 256)
                    a.o[r * a.o_stride + (x / D) * a.o_head_stride + x % D] = 0.f;
            r += gridDim.x;
            if (r < R) zl = as_const(a.seq_lens)[r];
        }
    }
};

template <int D, bool BF, bool UNI>
__device__ __forceinline__ void decode_body(const nc_paged_decode_args &a) {
    using X = Decode<D, BF, UNI>;
    // the waves' O, or the join's 256 x (4 columns, max, sum)
    __shared__ __attribute__((aligned(16))) float s_mem[4 * 16 * X::OP > 256 * 6 ? 4 * 16 * X::OP : 256 * 6];
    __shared__ float s_ml[4][16][2];
    __shared__ uint32_t s_word;
    const uint32_t lane = threadIdx.x & 63u;
    X x{a, lane, (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane & 15u, lane >> 4, X::WK * (4u >> a.wave_shift),
        reinterpret_cast<float (*)[16][X::OP]>(s_mem), s_ml, &s_word};
    x.run();
}

}  // namespace

// `_odd`: pages of any size; the others take sizes that are multiples of 16.
#define NC_DECODE(D, T, BF)                                                                                      \
    extern "C" __global__ __launch_bounds__(256, 3) void nc_paged_decode_d##D##T(const nc_paged_decode_args a) {  \
        decode_body<D, BF, true>(a);                                                                             \
    }                                                                                                            \
    extern "C" __global__ __launch_bounds__(256, 3) void nc_paged_decode_d##D##_odd##T(const nc_paged_decode_args a) { \
        decode_body<D, BF, false>(a);                                                                            \
    }
NC_DECODE(16, , false)
NC_DECODE(32, , false)
NC_DECODE(64, , false)
NC_DECODE(128, , false)
NC_DECODE(16, _bf16, true)
NC_DECODE(32, _bf16, true)
NC_DECODE(64, _bf16, true)
NC_DECODE(128, _bf16, true)
