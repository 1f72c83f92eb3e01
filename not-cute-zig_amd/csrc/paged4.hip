// paged4.hip — kernels of a smaller paged cache for MI355X (gfx950, wave64): rows into pages of 4 bits and back
// (nc_paged4_append, nc_paged4_read), single-token attention over them (nc_paged4_decode_*), attention that keeps its scores
// (nc_paged4_mass_*) and the weights by token out of those (nc_paged4_weights), and eviction by them (nc_paged4_select,
// nc_paged4_part_*, nc_paged4_move). The interface is described in include/notcute_paged4.h.

#include "paged_decode.h"

#include "paged4_args.h"

// -------------------------------------------------------------------------------------------------
// Rows into 4-bit pages: of every 32 values x of a row the scale 2^k, k the least with max |x| <= 7 2^k (then the largest is at
// most half a step off), and x 2^-k to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, halves to the even code. Both are
// exact arithmetic: the sum that finds k is one of integers, the product by a power of two. A thread takes 8 values of K and of V,
// four neighbouring lanes a group. Rows come in and go out at 16 bytes a lane, codes at 4, and the slots' loads stand beside the rows':
// what there is to move bounds both. 30000 rows of 8 heads of 64, at odd addresses: append 15.4 us, 5.0 TB/s, read 13.2 us, 5.9 TB/s (a
// large copy moves 4.8). Rows are stored past the caches, which need the room (14.6 us else, and the append behind it 21); codes, 4
// bytes a lane, are not (29.2 us for both, 34 with). One step of 16 requests is two launches' latency, 4.8 us for both. (2 or 4 rows a
// thread, a head's rows a workgroup, and blocks dealt to the XCDs in runs were no faster.)
// -------------------------------------------------------------------------------------------------
namespace {

typedef u32x4 __attribute__((aligned(2))) u32x4_loose;  // global memory takes 16 bytes at any alignment

__device__ __forceinline__ u32x4 load_eight(const uint16_t *p) {
    u32x4 r;
    __builtin_memcpy(&r, p, 16);  // one load: global memory takes them at any alignment
    return r;
}

// The largest over each 4 neighbouring lanes.
__device__ __forceinline__ uint32_t near_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, false));  // quad_perm 1,0,3,2 and 2,3,0,1
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, false));
}

// The lane's 8 codes, and its group's scale byte.
__device__ __forceinline__ uint32_t quantise(u32x4 w, bool bf, uint32_t &byte) {
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = w[i];  // a bit cast of a vector's element reads its first one
        const half2v h = __builtin_bit_cast(half2v, u);
        x[2 * i] = bf ? __uint_as_float(u << 16) : (float)h[0];
        x[2 * i + 1] = bf ? __uint_as_float(u & 0xffff0000u) : (float)h[1];
        top = max(top, max(__float_as_uint(x[2 * i]) & 0x7fffffffu, __float_as_uint(x[2 * i + 1]) & 0x7fffffffu));
    }
    top = near_max(top);
    const bool fine = top < 0x7f800000u;
    // 7 = 1.75 * 4: one more where the fraction is above 0.75
    const int e = (int)((top + 0x1fffffu) >> 23) - 2;
    const int b = min(max(e, bf ? NC_PAGED4_LEAST_BF16 : NC_PAGED4_LEAST_F16), bf ? NC_PAGED4_MOST_BF16 : NC_PAGED4_MOST_F16);
    byte = fine ? (uint32_t)b : 255u;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_ldexpf(x[i], 127 - b);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[0], x[1], 1.f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[2], x[3], 1.f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[4], x[5], 1.f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[6], x[7], 1.f, 3);
    return fine ? q : 0u;
}

// The value of 8 codes in the rows' type.
__device__ __forceinline__ u32x4 values(uint32_t q, uint32_t byte, bool bf) {
    const float s = __uint_as_float(byte << 23);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = pair_of_fours(q, s, i);
        const half2v h = {(_Float16)__uint_as_float(b << 16), (_Float16)__uint_as_float(b & 0xffff0000u)};
        r[i] = bf ? b : __builtin_bit_cast(uint32_t, h);
    }
    return r;
}

// Where a unit of 8 values of a row is: of the rows, and of the cache.
struct Place {
    uint64_t row, cache;
    bool in;
};
__device__ __forceinline__ Place place_of(const nc_paged4_rows_args &a, uint64_t row0, uint32_t u) {
    const uint32_t i = nc_paged_quot(u, a.chunks), c = u - i * a.chunks.d;
    const uint32_t h = c >> a.chunk_shift, x = c & ((1u << a.chunk_shift) - 1u);
    const uint32_t slot = (uint32_t)a.slots[row0 + i];
    Place p;
    p.in = slot < a.num_slots;
    const uint32_t page = nc_paged_quot(p.in ? slot : 0u, a.ps), t = (p.in ? slot : 0u) - page * a.ps.d;
    p.row = (row0 + i) * a.row_stride + h * a.row_head_stride + 8 * x;
    p.cache = page * a.page_stride + h * a.head_stride + t * a.token_stride + 8 * x;
    return p;
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void nc_paged4_append(const nc_paged4_rows_args a) {
    const uint64_t row0 = (uint64_t)blockIdx.x * a.wg_rows;
    const uint32_t rows = (uint32_t)min((uint64_t)a.wg_rows, a.num_rows - row0), total = rows * a.chunks.d;
    for (uint32_t u = threadIdx.x; u < total; u += blockDim.x) {
        const Place p = place_of(a, row0, u);
        const u32x4 kw = load_eight(a.k_in + p.row), vw = load_eight(a.v_in + p.row);  // on their way beside the slot
        if (!p.in) continue;  // all four lanes of a group
        uint32_t kb, vb;
        const uint32_t kq = quantise(kw, a.bf, kb), vq = quantise(vw, a.bf, vb);
        *reinterpret_cast<uint32_t *>(a.k + p.cache / 2) = kq;
        *reinterpret_cast<uint32_t *>(a.v + p.cache / 2) = vq;
        if (u % 4 == 0) {
            a.k_scales[p.cache / 32] = (uint8_t)kb;
            a.v_scales[p.cache / 32] = (uint8_t)vb;
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void nc_paged4_read(const nc_paged4_rows_args a) {
    const uint64_t row0 = (uint64_t)blockIdx.x * a.wg_rows;
    const uint32_t rows = (uint32_t)min((uint64_t)a.wg_rows, a.num_rows - row0), total = rows * a.chunks.d;
    for (uint32_t u = threadIdx.x; u < total; u += blockDim.x) {
        const Place p = place_of(a, row0, u);
        u32x4 k = {0u, 0u, 0u, 0u}, v = k;
        if (p.in) {
            const uint32_t kq = *reinterpret_cast<const uint32_t *>(a.k + p.cache / 2), vq = *reinterpret_cast<const uint32_t *>(a.v + p.cache / 2);
            k = values(kq, a.k_scales[p.cache / 32], a.bf);
            v = values(vq, a.v_scales[p.cache / 32], a.bf);
        }
        __builtin_nontemporal_store(k, reinterpret_cast<u32x4_loose *>(a.k_out + p.row));
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4_loose *>(a.v_out + p.row));
    }
}

// -------------------------------------------------------------------------------------------------
// Weights by token: mass[r][j] += sum over the query heads of exp2(score - max) / sum, out of the scores that an attention has
// kept. Four tokens a lane, every fourth head a wave; the waves' sums are added in their order. The scores are in the caches
// or were on their way out: 5 us for 16 requests of 4096 tokens and 32 heads (8.4 MB), 4.7 for 64 ragged ones.
// -------------------------------------------------------------------------------------------------
extern "C" __global__ __launch_bounds__(256) void nc_paged4_weights(const nc_paged_mass_args a) {
    __shared__ float s_sum[4][256];
    const uint32_t lane = threadIdx.x & 63u, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t r = blockIdx.y; r < a.num_seqs; r += gridDim.y) {
        const uint32_t len = nc_paged_cut(as_const(a.seq_lens)[r], a.max_tokens);
        for (uint32_t t0 = blockIdx.x * 256u; t0 < len; t0 += gridDim.x * 256u) {
            const uint32_t t = t0 + 4 * lane, j = t0 + threadIdx.x;
            const float old = j < len ? a.mass[r * a.mass_stride + j] : 0.f;  // on its way beside the scores
            floatx4 sum = {0.f, 0.f, 0.f, 0.f};
            if (t < len) {
                const uint64_t row0 = (uint64_t)r * a.num_q_heads;
#pragma unroll 8
                for (uint32_t h = w; h < a.num_q_heads; h += 4) {
                    const floatx4 s = *reinterpret_cast<const floatx4 *>(a.scores + (row0 + h) * a.score_pitch + t);
                    const float top = a.row_ml[2 * (row0 + h)], inv = a.row_ml[2 * (row0 + h) + 1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] += __builtin_amdgcn_exp2f(s[i] - top) * inv;
                }
            }
            *reinterpret_cast<floatx4 *>(&s_sum[w][4 * lane]) = sum;
            __syncthreads();
            if (j < len) a.mass[r * a.mass_stride + j] = old + (s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x] + s_sum[2][threadIdx.x] + s_sum[3][threadIdx.x]);
            __syncthreads();
        }
    }
}

// -------------------------------------------------------------------------------------------------
// Eviction: select, then move. The least mass that is kept is found by its bits, 11 at a time from the top (a histogram of the
// masses that agree in the bits above, until all of a bin are kept); then the tokens that stay are listed, in their order. Masses are read
// once into registers as far as they fit, and what is left is a chain of barriers, loads and LDS additions in code that runs once:
//   by one workgroup a request, of 8 waves with 2 tokens a lane (tables of up to 2048 tokens) or of 16 with 8;
//   by parts in four launches, for tables of 12288 tokens and more.
// With the rows' move, in replayed graphs and with fresh masses, over 2 heads of 64, half the tokens kept:
//   requests x tokens    8 waves   16 waves   parts
//   1 x 300                 9.6      12.3      15.9 us
//   1 x 1000               12.4      15.3      18.2
//   200 x 2000             61.0      63.8      69.5
//   16 x 4097              26.8      25.6      30.9
//   1 x 8000               25.4      21.0      21.3
//   16 x 8000              39.7      34.9      38.0
//   4 x 16000              52.5      39.3      34.5
//   100 x 16000             221       207       224 (by parts all the same: more often a few of them are cut)
//   1 x 60000               143      84.8      45.2
// What bounds short ones is that chain (6.8 us of selection for 300 tokens, 9 for 200 requests of 1001), long ones the four launches of
// 5 to 12 us, and large moves the rate of a copy.
// -------------------------------------------------------------------------------------------------
namespace {

// Masses in ascending order as numbers: both zeros are one, a NaN is the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 + 0 is 0
    return x != x ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, nc_paged_div ps) {
    const uint32_t n = nc_paged_quot(tokens, ps);
    return n + (n * ps.d != tokens);
}

// A barrier of waves that only exchange what is in LDS: their stores to memory need not have arrived.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ uint32_t lanes_below(uint64_t who) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
}

// The mass of an order.
__device__ __forceinline__ float mass_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }

// What is kept of the tokens that are neither first nor last: all masses above `edge` (all_nan: no such), and the first `ties` tokens
// of that mass.
struct Edge {
    float edge;
    uint32_t ties;
    bool all_nan;
};
// From the bits of orders down to `shift`: `whole`, all of those with these bits are kept, so that the edge is the order below
// the least of them; else all bits are known, and `left` of those are kept. Orders that no mass has: below 0's, whose mass would be -0, and
// between infinity's and NaN's. (Below -infinity's the mass is a NaN, above which is everything.)
__device__ __forceinline__ Edge edge_of(uint32_t prefix, int shift, bool whole, uint32_t left) {
    uint32_t order = prefix;
    if (whole) {
        order = prefix << shift;
        order -= order != 0u;
        order = order == 0x7fffffffu ? 0x7ffffffeu : min(order, 0xff800000u);
    }
    return {mass_of(order), whole ? 0u : left, order == 0xffffffffu};
}

constexpr uint32_t kBins = NC_PAGED4_BINS;

// A workgroup's tokens of a request, begin..end-1 of them a wave's. HELD: tokens that a lane keeps, and of others reads at once.
template <uint32_t WAVES, uint32_t HELD>
struct Tokens {
    static constexpr uint32_t THREADS = 64 * WAVES;
    static constexpr uint32_t EACH = kBins / THREADS;  // bins of a thread
    // Equal masses are LDS additions to one address, one after the other: every bin COPIES times, a lane to its own. (60001 tokens of
    // few different masses, by one workgroup: 59 us with one.)
    static constexpr uint32_t COPIES = WAVES == 16 ? 8 : 2;

    const nc_paged_evict_args &a;
    const uint32_t r, n, tid, lane, w, lo, hi, need;
    const float *mass;
    const int32_t *row;
    uint32_t begin, end;
    float held_mass[HELD];
    uint32_t held_page[HELD];

    __device__ __forceinline__ Tokens(const nc_paged_evict_args &args, uint32_t request, uint32_t len, uint32_t wave)
        : a(args), r(request), n(len), tid(threadIdx.x), lane(threadIdx.x & 63u), w(wave), lo(args.sinks), hi(len - args.recent),
          need(args.budget - args.sinks - args.recent), mass(args.mass + request * args.mass_stride), row(args.table + request * args.table_stride) {}

    // Those of `from`..`from + 64 * WAVES * x - 1` that there are, shared out among the waves.
    __device__ __forceinline__ void take(uint32_t from, uint32_t tokens, bool there, bool pages) {
        const uint32_t part = (tokens + 64u * WAVES - 1u) / (64u * WAVES) * 64u, stop = min(from + tokens, n);
        begin = min(from + w * part, stop);
        end = min(begin + part, stop);
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i) {
            const uint32_t t = begin + 64u * i + lane;
            held_mass[i] = there && t < end ? mass[t] : 0.f;
            held_page[i] = there && pages && t < end ? (uint32_t)row[nc_paged_quot(t, a.ps)] : 0u;
        }
    }

    // fn(64 neighbours' first place, the lane's mass) for all of the wave's tokens; those that are not in registers so many read at once.
    template <class F>
    __device__ __forceinline__ void each(F &&fn) const {
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i)
            if (begin + 64u * i < end) fn(begin + 64u * i, held_mass[i]);
        for (uint32_t t0 = begin + 64u * HELD; t0 < end; t0 += 64u * HELD) {
            float x[HELD];
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i) x[i] = t0 + 64u * i + lane < end ? mass[t0 + 64u * i + lane] : 0.f;
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i)
                if (t0 + 64u * i < end) fn(t0 + 64u * i, x[i]);
        }
    }

    // Sums over the waves' numbers: of all of them, or of those before this one.
    __device__ __forceinline__ uint32_t sum_of(const uint32_t *sums, uint32_t waves) const {
        const uint32_t scan = wave_scan32(lane < waves ? sums[lane] : 0u);
        return (uint32_t)__builtin_amdgcn_readlane(scan, 63);
    }

    // Counts, by `bits` bits from `shift` on, of the orders that have `prefix` above those.
    __device__ __forceinline__ void count(uint32_t *bins, uint32_t prefix, int shift, int bits) const {
        for (uint32_t i = tid; i < kBins * COPIES; i += THREADS) bins[i] = 0;
        lds_barrier();
        each([&](uint32_t t0, float x) {
            const uint32_t t = t0 + lane, k = order_of(x);
            const bool mine = t >= lo && t < hi && t < end && (shift == 21 || k >> (shift + bits) == prefix);
            const uint32_t bin = k >> shift & ((1u << bits) - 1u);
            if (mine) atomicAdd(&bins[bin * COPIES + lane % COPIES], 1u);
        });
        lds_barrier();
    }
    // Bin 2047 - EACH * tid - i.
    __device__ __forceinline__ uint32_t bin_of(const uint32_t *bins, uint32_t i) const {
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t x = 0; x < COPIES; ++x) sum += bins[(kBins - 1u - EACH * tid - i) * COPIES + x];
        return sum;
    }

    // Pages that become free: to the list, behind those of the requests before this one; which requests are cut, and the totals.
    __device__ __forceinline__ void sums(bool cut, uint32_t keep, uint32_t (*s_sums)[WAVES]) const {
        if (cut && a.chunks > 1) {
            for (uint32_t i = tid; i < a.chains; i += THREADS) a.taken[(uint64_t)r * a.chains + i] = 0;
            for (uint32_t i = tid; i < a.chains * a.chunks; i += THREADS) a.read[(uint64_t)r * a.chains * a.chunks + i] = 0;
        }
        uint32_t x[5] = {0, 0, 0, 0, 0};  // pages of all, and of those before this one; requests cut, and before; tokens
        for (uint32_t q = tid; q < a.num_seqs; q += THREADS) {
            const uint32_t m = nc_paged_cut(a.seq_lens[q], a.max_tokens);
            if (m > a.limit) {
                const uint32_t f = pages_of(m, a.ps) - pages_of(a.budget, a.ps);
                x[0] += f;
                x[1] += q < r ? f : 0u;
                x[2] += 1u;
                x[3] += q < r ? 1u : 0u;
                x[4] += m - a.budget;
            }
        }
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            x[i] = wave_scan32(x[i]);
            if (lane == 63) s_sums[i][w] = x[i];
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < 5; ++i) x[i] = sum_of(s_sums[i], WAVES);
        const int64_t base = (int64_t)a.cursor[0] - x[0];
        if (r == 0 && tid == 0) {
            a.totals[0] = (int32_t)max(base, (int64_t)0);  // for counts[0], which may be the cursor that others read
            a.totals[1] = (int32_t)x[2];
            a.counts[1] = (int32_t)x[2];
            a.counts[2] = (int32_t)x[0];
            a.counts[3] = (int32_t)x[4];
        }
        if (!cut) return;
        if (tid == 0) a.cuts[x[3]] = (int32_t)r;
        const uint32_t held = pages_of(n, a.ps), stay = pages_of(keep, a.ps);
        for (uint32_t p = stay + tid; p < held; p += THREADS) {
            const int64_t at = base + x[1] + (p - stay);
            if (at >= 0 && at < (int64_t)a.free_len) a.free_pages[at] = row[p];
        }
    }

    // Lists the tokens that stay, behind `sure` that stay for sure and `last` of the edge's mass. The least that goes.
    __device__ __forceinline__ uint32_t list(const Edge &e, uint32_t sure, uint32_t last, uint32_t *s_a, uint32_t *s_b) const {
        // Which of 64 neighbours stay for sure, and which have the edge's mass. (A NaN is above every number.)
        auto sure_of = [&](uint32_t t0, float x) {
            const bool above = !e.all_nan && !(x <= e.edge);
            if (t0 >= lo && t0 + 64u <= hi) return __ballot(above);
            const uint32_t t = t0 + lane;
            return __ballot(t < end && (t < lo || t >= hi || above));
        };
        auto last_of = [&](uint32_t t0, float x) {
            const bool equal = e.all_nan ? x != x : x == e.edge;
            const uint32_t t = t0 + lane;
            return t0 >= lo && t0 + 64u <= hi ? __ballot(equal) : __ballot(equal && t >= lo && t < hi && t < end);
        };
        uint32_t ws = 0, wl = 0;
        each([&](uint32_t t0, float x) {
            ws += __builtin_popcountll(sure_of(t0, x));
            if (e.ties) wl += __builtin_popcountll(last_of(t0, x));
        });
        lds_barrier();
        if (lane == 0) {
            s_a[w] = ws;
            s_b[w] = wl;
        }
        lds_barrier();
        sure += sum_of(s_a, w);
        last += sum_of(s_b, w);
        int32_t *source = a.source + (uint64_t)r * a.max_tokens;
        float *kept = a.kept_mass + (uint64_t)r * a.max_tokens;
        uint32_t gone = n;
        // The place in its page of the lane's token of 64 neighbours, who are listed one after the other.
        const uint32_t at64 = nc_paged_quot(64u, a.ps), tok64 = 64u - at64 * a.ps.d;
        uint32_t tok = begin + lane - nc_paged_quot(begin + lane, a.ps) * a.ps.d;
        auto put = [&](uint32_t t0, float x, uint32_t page) {
            const uint32_t t = t0 + lane;
            const uint64_t who = sure_of(t0, x), tie = e.ties ? last_of(t0, x) : 0ull;
            const uint32_t nl = last + lanes_below(tie), to = sure + lanes_below(who) + min(nl, e.ties);
            const bool stays = who >> lane & 1ull || (tie >> lane & 1ull && nl < e.ties);
            if (stays && to < a.budget) {  // as it is, unless something changes the masses meanwhile
                source[to] = page < a.num_pages ? (int32_t)(page * a.ps.d + tok) : -1;
                kept[to] = x;
            } else if (!stays && t < end) {
                gone = min(gone, t);
            }
            tok += tok64;
            tok -= tok >= a.ps.d ? a.ps.d : 0u;
            sure += __builtin_popcountll(who);
            last += __builtin_popcountll(tie);
        };
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i)
            if (begin + 64u * i < end) put(begin + 64u * i, held_mass[i], held_page[i]);
        for (uint32_t t0 = begin + 64u * HELD; t0 < end; t0 += 64u * HELD) {
            float x[HELD];
            uint32_t page[HELD];
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i) {
                const uint32_t t = min(t0 + 64u * i + lane, n - 1u);
                x[i] = mass[t];
                page[i] = (uint32_t)row[nc_paged_quot(t, a.ps)];
            }
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i)
                if (t0 + 64u * i < end) put(t0 + 64u * i, x[i], page[i]);
        }
        return gone;
    }
};

// All of a request by one workgroup.
template <uint32_t WAVES, uint32_t HELD>
__device__ __forceinline__ void select_body(const nc_paged_evict_args &a) {
    using T = Tokens<WAVES, HELD>;
    __shared__ uint32_t s_bins[kBins * T::COPIES];
    __shared__ uint32_t s_sums[5][WAVES];
    __shared__ uint32_t s_bin, s_above, s_count, s_first;
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const uint32_t n = nc_paged_cut(as_const(a.seq_lens)[r], a.max_tokens);
    const bool cut = n > a.limit;
    const uint32_t keep = cut ? a.budget : n;
    if (tid == 0) {
        a.news[r] = (int32_t)keep;
        a.olds[r] = (int32_t)n;
        s_first = n;
    }
    if (!cut && r != 0) return;
    T x(a, r, n, __builtin_amdgcn_readfirstlane(tid >> 6));
    x.take(0, n, cut, true);
    x.sums(cut, keep, s_sums);
    if (!cut) return;
    Edge e = {__builtin_inff(), 0u, true};
    if (x.need) {
        uint32_t prefix = 0, left = x.need;  // the bits above the present ones, kept tokens that agree in them
        for (int shift = 21, bits = 11;;) {
            x.count(s_bins, prefix, shift, bits);
            // Bins from the top, EACH a thread; the one that the last token to be kept is in.
            uint32_t bin[T::EACH], mine = 0;
#pragma unroll
            for (uint32_t i = 0; i < T::EACH; ++i) mine += bin[i] = x.bin_of(s_bins, i);
            const uint32_t incl = wave_scan32(mine);
            if (x.lane == 63) s_sums[0][x.w] = incl;
            lds_barrier();
            uint32_t above = incl - mine + x.sum_of(s_sums[0], x.w);
            if (above < left && left <= above + mine) {
#pragma unroll
                for (uint32_t i = 0; i < T::EACH; ++i) {
                    if (above < left && left <= above + bin[i]) {
                        s_bin = kBins - 1u - T::EACH * tid - i;
                        s_above = above;
                        s_count = bin[i];
                    }
                    above += bin[i];
                }
            }
            lds_barrier();
            prefix = prefix << bits | s_bin;
            left -= s_above;
            if (s_count == left || shift == 0) {
                e = edge_of(prefix, shift, s_count == left, left);
                break;
            }
            bits = shift == 21 ? 11 : 10;
            shift = shift == 21 ? 10 : 0;
            lds_barrier();
        }
    }
    const uint32_t gone = x.list(e, 0, 0, s_sums[0], s_sums[1]);
    if (gone < n) atomicMin(&s_first, gone);
    lds_barrier();
    if (tid == 0) a.first[r] = (int32_t)s_first;
}

// A long request by several workgroups, `part` tokens each, in four launches: three that count, and one that lists. Each part leaves its
// counts, and every workgroup of the next launch adds up all of the request's (64 parts at most), and those before its own, which says
// where what it lists begins.
constexpr uint32_t PART_WAVES = 8, PART_HELD = 4;

// What a launch has found: the bits so far, kept tokens among those that agree in them, and whether that is all of them (`whole`, at
// `shift`).
struct PartState {
    uint32_t prefix, left, whole, shift;
};

template <int PASS>
__device__ __forceinline__ void part_body(const nc_paged_evict_args &a) {
    using T = Tokens<PART_WAVES, PART_HELD>;
    static_assert(T::EACH == 4, "a thread's bins are one load");
    __shared__ uint32_t s_bins[PASS < 4 ? kBins * T::COPIES : 1];
    __shared__ uint32_t s_sums[5][PART_WAVES];
    __shared__ uint32_t s_bin, s_above, s_count, s_low, s_low_at, s_first;
    const uint32_t wgs = a.parts + (PASS == 1), r = blockIdx.x / wgs, p = blockIdx.x - r * wgs, tid = threadIdx.x;
    const uint32_t n = nc_paged_cut(as_const(a.seq_lens)[r], a.max_tokens);
    const bool cut = n > a.limit;
    T x(a, r, n, __builtin_amdgcn_readfirstlane(tid >> 6));
    if (PASS == 1 && p == a.parts) {  // beside the parts'
        const uint32_t keep = cut ? a.budget : n;
        if (tid == 0) {
            a.news[r] = (int32_t)keep;
            a.olds[r] = (int32_t)n;
            a.first[r] = (int32_t)n;
        }
        if (cut || r == 0) x.sums(cut, keep, s_sums);
        return;
    }
    const uint32_t from = p * a.part;
    if (!cut || from >= n || (PASS < 4 && !x.need)) return;
    x.take(from, a.part, true, PASS == 4);
    const uint32_t parts = (n - 1u) / a.part + 1u;
    PartState *states = reinterpret_cast<PartState *>(a.states) + 2 * (uint64_t)r;  // of passes 2 and 3
    uint32_t *lows = a.lows + 2 * ((uint64_t)r * a.parts + p);                       // kept ones in the parts before this one
    // Passes 1 and 3 leave their counts in one place, pass 2 in another.
    auto counts_of = [&](int pass) { return (pass == 2 ? a.counts2 : a.counts1) + (uint64_t)r * a.parts * kBins; };

    PartState state = {0u, x.need, 0u, 21u};
    uint32_t low = 0, low_at = 0;
    if (PASS > 2 && x.need) {
        state = states[PASS > 2 ? PASS - 3 : 0];
        low = lows[PASS > 2 ? PASS - 3 : 0];
    }
    if (PASS > 1 && x.need && !state.whole) {
        const uint32_t *counts = counts_of(PASS - 1);
        u32x4 all = {0u, 0u, 0u, 0u}, before = all;  // bins 2044 - 4 tid.., of all parts and of those before this one
        const uint32_t at = kBins - 4u - 4u * tid;
#pragma unroll 8
        for (uint32_t q = 0; q < parts; ++q) {
            const u32x4 y = *reinterpret_cast<const u32x4 *>(counts + (uint64_t)q * kBins + at);
            all += y;
            if (q < p) before += y;
        }
        const uint32_t mine = all[0] + all[1] + all[2] + all[3], mine_low = before[0] + before[1] + before[2] + before[3];
        const uint32_t incl = wave_scan32(mine), incl_low = wave_scan32(mine_low);
        if (x.lane == 63) {
            s_sums[0][x.w] = incl;
            s_sums[1][x.w] = incl_low;
        }
        lds_barrier();
        uint32_t above = incl - mine + x.sum_of(s_sums[0], x.w), lower = incl_low - mine_low + x.sum_of(s_sums[1], x.w);
        if (above < state.left && state.left <= above + mine) {
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                if (above < state.left && state.left <= above + all[i]) {
                    s_bin = at + i;
                    s_above = above;
                    s_count = all[i];
                    s_low = lower;
                    s_low_at = before[i];
                }
                above += all[i];
                lower += before[i];
            }
        }
        lds_barrier();
        state.shift = PASS == 2 ? 21u : PASS == 3 ? 10u : 0u;
        state.prefix = state.prefix << (PASS == 4 ? 10 : 11) | s_bin;
        state.left -= s_above;
        state.whole = s_count == state.left;
        low += s_low + (state.whole ? s_low_at : 0u);
        low_at = state.whole ? 0u : s_low_at;
    }
    if constexpr (PASS < 4) {
        if constexpr (PASS > 1) {
            if (tid == 0) {
                if (p == 0) states[PASS - 2] = state;
                lows[PASS - 2] = low;
            }
            if (state.whole) return;
        }
        x.count(s_bins, state.prefix, PASS == 1 ? 21 : PASS == 2 ? 10 : 0, PASS == 3 ? 10 : 11);
        u32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = x.bin_of(s_bins, 3 - i);
        *reinterpret_cast<u32x4 *>(counts_of(PASS) + (uint64_t)p * kBins + kBins - 4u - 4u * tid) = y;
    } else {
        const Edge e = x.need ? edge_of(state.prefix, (int)state.shift, state.whole, state.left) : Edge{__builtin_inff(), 0u, true};
        if (tid == 0) s_first = n;
        const uint32_t gone = x.list(e, low + min(from, x.lo) + (from > x.hi ? from - x.hi : 0u), low_at, s_sums[2], s_sums[3]);
        if (gone < n) atomicMin(&s_first, gone);
        lds_barrier();
        if (tid == 0 && s_first < n) atomicMin(reinterpret_cast<uint32_t *>(a.first) + r, s_first);
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(1024) void nc_paged4_select(const nc_paged_evict_args a) { select_body<16, 8>(a); }
extern "C" __global__ __launch_bounds__(512) void nc_paged4_select_short(const nc_paged_evict_args a) { select_body<8, 2>(a); }
extern "C" __global__ __launch_bounds__(64 * PART_WAVES) void nc_paged4_part_first(const nc_paged_evict_args a) { part_body<1>(a); }
extern "C" __global__ __launch_bounds__(64 * PART_WAVES) void nc_paged4_part_second(const nc_paged_evict_args a) { part_body<2>(a); }
extern "C" __global__ __launch_bounds__(64 * PART_WAVES) void nc_paged4_part_third(const nc_paged_evict_args a) { part_body<3>(a); }
extern "C" __global__ __launch_bounds__(64 * PART_WAVES) void nc_paged4_part_list(const nc_paged_evict_args a) { part_body<4>(a); }

// The rows that stay, to the front, in place and all at once. A chunk's workgroup reads its rows, says so, and stores them when the
// chunks before it in the chain have been read: a place holds a row that goes to itself or to a place before it. Chunks are
// taken by a count, in their order, and reading waits for nothing, so whoever waits does so for workgroups that run; that needs no
// order among workgroups, and not all of them at once.
// Stores go past the caches. 16 requests of 4097 tokens cut to 2048, 8 heads of 128: 52 us, 5.2 TB/s read and written (through the caches
// 60); with the selection 67.5 us, one of 60000 104. (A wave a column that walks down the rows, which needs no flags: 100 and 346 us.)
namespace {

// A store that is asked for has been seen by whoever reads the flag: waits as in Decode::join(). False where the tries, some tenth of
// a second's, ended the wait: the workspace was not this call's alone.
__device__ __forceinline__ bool wait_for_chunks(const uint32_t *read, uint32_t chunk, uint32_t most_tries) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t c0 = 0; c0 < chunk; c0 += 64) {
        bool all = false;
        for (uint32_t tries = 0; tries < most_tries && !all; ++tries) {
            if (tries) __builtin_amdgcn_s_sleep(2);
            all = __all(c0 + lane >= chunk || __hip_atomic_load(read + c0 + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0u);
        }
        if (!all) return false;
    }
    return true;
}

template <bool FOUR>
__device__ __forceinline__ void move_chunk(const nc_paged_evict_args &a, uint32_t r, uint32_t chain, uint32_t chunk, uint32_t keep, uint32_t first,
                                           uint32_t *read, uint32_t *s_late) {
    constexpr uint32_t ROWS = NC_PAGED4_MOVE_ROWS;
    constexpr uint32_t UE = FOUR ? 32 : 8;  // values of a unit
    const uint32_t tid = threadIdx.x, at_once = NC_PAGED4_MOVE_THREADS >> a.row_log2;
    const uint32_t v = chain & 1u, unit = tid & ((1u << a.row_log2) - 1u);
    const uint32_t head = ((chain >> 1) << (a.row_log2 - a.unit_log2)) + (unit >> a.unit_log2);
    const uint64_t base = head * a.head_stride + UE * (unit & ((1u << a.unit_log2) - 1u));
    uint8_t *codes = v ? a.v : a.k, *scales = v ? a.v_scales : a.k_scales;
    const int32_t *row = a.table + r * a.table_stride, *source = a.source + (uint64_t)r * a.max_tokens;
    const uint32_t num_slots = a.num_pages * a.ps.d, j0 = first + chunk * (ROWS * at_once) + (tid >> a.row_log2);
    uint32_t slot[ROWS], page[ROWS];
#pragma unroll
    for (uint32_t i = 0; i < ROWS; ++i) {
        const uint32_t j = j0 + i * at_once, jj = min(j, keep - 1u);
        slot[i] = j < keep ? (uint32_t)source[jj] : ~0u;
        page[i] = (uint32_t)row[nc_paged_quot(jj, a.ps)];
    }
    u32x4 x[ROWS];
    uint32_t s[ROWS];
    bool in[ROWS];
#pragma unroll
    for (uint32_t i = 0; i < ROWS; ++i) {
        in[i] = slot[i] < num_slots && page[i] < a.num_pages;
        const uint32_t from = in[i] ? slot[i] : 0u, p = nc_paged_quot(from, a.ps);
        const uint64_t src = p * a.page_stride + (from - p * a.ps.d) * a.token_stride + base;
        x[i] = *reinterpret_cast<const u32x4 *>(codes + (FOUR ? src / 2 : src * 2));
        if constexpr (FOUR) s[i] = scales[src / 32];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (a.chunks > 1) {
        if (tid == 0) __hip_atomic_store(read + chunk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (chunk) {
            if (tid < 64) {
                const bool there = wait_for_chunks(read, chunk, a.tries);
                if (tid == 0) *s_late = !there;
            }
            __syncthreads();
            if (*s_late) {  // stored, these rows might be where others have still to be read
                if (tid == 0) __hip_atomic_store(a.counts + 1, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                return;
            }
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < ROWS; ++i)
        if (in[i]) {
            const uint32_t j = j0 + i * at_once, tok = j - nc_paged_quot(j, a.ps) * a.ps.d;
            const uint64_t to = page[i] * a.page_stride + tok * a.token_stride + base;
            __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4 *>(codes + (FOUR ? to / 2 : to * 2)));
            if constexpr (FOUR) scales[to / 32] = (uint8_t)s[i];
        }
}

}  // namespace

// What the selection left of the k-th request that is cut. It is held to what there is, so that a workspace that another call
// changes meanwhile costs a wrong result and nothing else.
struct Cut {
    uint32_t r, old, keep, first;
};
__device__ __forceinline__ Cut cut_of(const nc_paged_evict_args &a, uint32_t k) {
    Cut c;
    c.r = min((uint32_t)as_const(a.cuts)[k], a.num_seqs - 1u);
    c.old = min((uint32_t)as_const(a.olds)[c.r], a.max_tokens);
    c.keep = min((uint32_t)as_const(a.news)[c.r], c.old);
    c.first = min((uint32_t)as_const(a.first)[c.r], c.keep);
    return c;
}

extern "C" __global__ __launch_bounds__(NC_PAGED4_MOVE_THREADS) void nc_paged4_move(const nc_paged_evict_args a) {
    __shared__ uint32_t s_chunk, s_late;
    const uint32_t cuts = min((uint32_t)as_const(a.totals)[1], a.num_seqs);
    if (blockIdx.x < a.mass_wgs) {  // what else the selection left
        if (blockIdx.x == 0 && threadIdx.x == 0) a.counts[0] = a.totals[0];
        for (uint32_t r = blockIdx.x * NC_PAGED4_MOVE_THREADS + threadIdx.x; r < a.num_seqs; r += a.mass_wgs * NC_PAGED4_MOVE_THREADS) a.kept_lens[r] = a.news[r];
        for (uint64_t p = blockIdx.x; p < (uint64_t)cuts * a.mass_parts; p += a.mass_wgs) {
            const uint32_t k = (uint32_t)(p / a.mass_parts);
            const Cut c = cut_of(a, k);
            const uint32_t lo = (uint32_t)(p - (uint64_t)k * a.mass_parts) * NC_PAGED4_MASS_PART, end = min(lo + NC_PAGED4_MASS_PART, c.old);
            float *mass = a.mass + c.r * a.mass_stride;
            const float *kept = a.kept_mass + (uint64_t)c.r * a.max_tokens;
            for (uint32_t t = lo + threadIdx.x; t < end; t += NC_PAGED4_MOVE_THREADS)
                if (t >= c.first) mass[t] = t < c.keep ? kept[t] : 0.f;
        }
        return;
    }
    const uint32_t b = blockIdx.x - a.mass_wgs, all = cuts * a.chains;
    for (uint32_t q = b % a.side_chains; q < all; q += a.side_chains) {
        const uint32_t k = q / a.chains, chain = q - k * a.chains, size = nc_paged4_chunk(a.row_log2);
        const Cut c = cut_of(a, k);
        const uint32_t chunks = min((c.keep - c.first + size - 1u) / size, a.chunks);
        const uint64_t at = (uint64_t)c.r * a.chains + chain;
        while (true) {
            uint32_t chunk = 0;
            if (a.chunks > 1) {
                if (threadIdx.x == 0) s_chunk = __hip_atomic_fetch_add(a.taken + at, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __syncthreads();
                chunk = __builtin_amdgcn_readfirstlane(s_chunk);
                __syncthreads();
            }
            if (chunk >= chunks) break;
            if (a.four)
                move_chunk<true>(a, c.r, chain, chunk, c.keep, c.first, a.read + at * a.chunks, &s_late);
            else
                move_chunk<false>(a, c.r, chain, chunk, c.keep, c.first, a.read + at * a.chunks, &s_late);
            if (a.side_chunks >= a.chunks) break;  // every chunk has a workgroup
        }
    }
}

// -------------------------------------------------------------------------------------------------
// Attention: paged_decode.h.
// -------------------------------------------------------------------------------------------------
#define NC_DECODE4_KERNEL(NAME, D, BF, UNI, MANY, NEXT, FOUR, MASS, PACK)                               \
    extern "C" __global__ __launch_bounds__(64 * NC_PAGED_WAVES, 2) void NAME(const nc_paged_more_args) { \
        decode_body<D, BF, UNI, MANY, NEXT, FOUR, MASS, PACK>();                                        \
    }
#define NC_DECODE4_PACK(D, T, PACK, NEXT)                                                        \
    NC_DECODE4_KERNEL(nc_paged4_decode_d##D##T, D, true, true, true, NEXT, true, false, PACK)        \
    NC_DECODE4_KERNEL(nc_paged4_decode_d##D##T##_odd, D, true, false, true, NEXT, true, false, PACK) \
    NC_DECODE4_KERNEL(nc_paged4_mass4_d##D##T, D, true, true, true, NEXT, true, true, PACK)          \
    NC_DECODE4_KERNEL(nc_paged4_mass4_d##D##T##_odd, D, true, false, true, NEXT, true, true, PACK)
#define NC_DECODE4(D)                 \
    NC_DECODE4_PACK(D, , 1, false)    \
    NC_DECODE4_PACK(D, _by2, 2, true) \
    NC_DECODE4_PACK(D, _by4, 4, true)
NC_DECODE4(32)
NC_DECODE4(64)
NC_DECODE4(128)
// Scores kept over caches in 16 bits.
#define NC_MASS(D, T, BF)                                                                  \
    NC_DECODE4_KERNEL(nc_paged4_mass_d##D##T, D, BF, true, false, false, false, true, 1)           \
    NC_DECODE4_KERNEL(nc_paged4_mass_d##D##_odd##T, D, BF, false, false, false, false, true, 1)
NC_MASS(16, , false)
NC_MASS(32, , false)
NC_MASS(64, , false)
NC_MASS(128, , false)
NC_MASS(16, _bf16, true)
NC_MASS(32, _bf16, true)
NC_MASS(64, _bf16, true)
NC_MASS(128, _bf16, true)
