// paged.hip — the paged key-value cache's kernels for MI355X (gfx950, wave64): block tables and slot map
// (nc_paged_build), row append (nc_paged_append_*) and single-token attention (nc_paged_decode_*). The
// interface is described in include/notcute_paged.h. What device memory names (lengths, page ids, slots) is
// checked here before it becomes an address.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_args.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

template <bool BF>
__device__ __forceinline__ float to_f32(uint16_t h) {
    if constexpr (BF)
        return __uint_as_float((uint32_t)h << 16);
    else
        return (float)__builtin_bit_cast(_Float16, h);
}

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
// Single-token attention: one workgroup per request and query head, its waves taking every fourth key.
// -------------------------------------------------------------------------------------------------
namespace {

template <int D, bool BF>
__device__ __forceinline__ void decode_body(const nc_paged_decode_args &a) {
    constexpr int E = (D + 63) / 64;  // dims of a lane
    __shared__ float s_o[4][D], s_ml[4][2];
    const uint32_t r = blockIdx.x / a.num_q_heads, head = blockIdx.x % a.num_q_heads, kh = head / a.group;
    const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
    const uint32_t len = nc_paged_cut(a.seq_lens[r], a.max_tokens);
    const float sc = a.scale * kLog2e;
    float q[E], acc[E] = {}, m = neg_inf(), l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t c = lane + 64 * e;
        q[e] = c < D ? to_f32<BF>(a.q[r * a.q_stride + head * a.q_head_stride + c]) : 0.f;
    }
    for (uint32_t j = w; j < len; j += 4) {
        const uint32_t at = nc_paged_quot(j, a.ps);
        const uint32_t page = (uint32_t)a.table[r * a.table_stride + at];
        if (page >= a.num_pages) continue;
        const uint64_t base = page * a.page_stride + kh * a.head_stride + (j - at * a.ps.d) * a.token_stride;
        float s = 0.f, v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t c = lane + 64 * e;
            v[e] = c < D ? to_f32<BF>(a.v[base + c]) : 0.f;
            s += q[e] * (c < D ? to_f32<BF>(a.k[base + c]) : 0.f);
        }
#pragma unroll
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x, 64);
        s *= sc;
        const float mn = fmaxf(m, s), base_m = mn == neg_inf() ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - base_m), p = __builtin_amdgcn_exp2f(s - base_m);
        l = l * alpha + p;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * alpha + p * v[e];
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < D) s_o[w][lane + 64 * e] = acc[e];
    if (lane == 0) {
        s_ml[w][0] = m;
        s_ml[w][1] = l;
    }
    __syncthreads();
    if (threadIdx.x < D) {
        float top = neg_inf(), sum = 0.f, o = 0.f;
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s_ml[i][0]);
        if (top == neg_inf()) top = 0.f;
        for (int i = 0; i < 4; ++i) {
            const float f = __builtin_amdgcn_exp2f(s_ml[i][0] - top);
            sum += f * s_ml[i][1];
            o += f * s_o[i][threadIdx.x];
        }
        a.o[r * a.o_stride + head * a.o_head_stride + threadIdx.x] = sum == 0.f ? 0.f : o / sum;
    }
}

}  // namespace

#define NC_DECODE(D, T, BF)                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void nc_paged_decode_d##D##T(const nc_paged_decode_args a) {    \
        decode_body<D, BF>(a);                                                                                  \
    }
NC_DECODE(16, , false)
NC_DECODE(32, , false)
NC_DECODE(64, , false)
NC_DECODE(128, , false)
NC_DECODE(16, _bf16, true)
NC_DECODE(32, _bf16, true)
NC_DECODE(64, _bf16, true)
NC_DECODE(128, _bf16, true)
