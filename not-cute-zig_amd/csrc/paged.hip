// paged.hip — the paged key-value cache's kernels for MI355X (gfx950, wave64): block tables and slot map
// (nc_paged_build), row append (nc_paged_append_*) and single-token attention (nc_paged_decode_*). The
// interface is described in include/notcute_paged.h. What device memory names (lengths, page ids, slots) is
// checked here before it becomes an address.

#include "paged_decode.h"

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
