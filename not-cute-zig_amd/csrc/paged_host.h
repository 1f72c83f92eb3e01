// paged_host.h — host side that paged.cpp and paged4.cpp share: options, overlaps of tensors, the attention's plan and launch.
// Nothing here allocates or synchronises.
#ifndef NOTCUTE_PAGED_HOST_H
#define NOTCUTE_PAGED_HOST_H

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "notcute_paged.h"
#include "paged_args.h"

extern "C" int nc_internal_fail(int status, const char *what);
// hip_api.cpp: a function of the module, looked up once and kept under `slot` (of paged.hip's kernels, then paged4.hip's).
extern "C" int nc_internal_module_kept_function(nc_module module, uint32_t slot, const char *name, nc_function *out);

namespace nc_paged {

constexpr uint64_t kMost31 = 0x7fffffffull;
constexpr uint64_t kMostUnits = 1ull << 30;
constexpr uint64_t kMostElements = 1ull << 60;

// The options with every stride resolved.
struct Shape {
    nc_paged_options o;
    uint64_t group, cache_len, table_len, q_len, o_len;
    uint64_t heads, seq_units;  // the attention's: key heads (parts of them), and most units of a head
};

inline uint64_t or_packed(uint64_t stride, uint64_t count, uint64_t inner) { return stride ? stride : count * inner; }

struct Axis {
    uint64_t n, stride;
};

// Elements from a tensor's first to behind its last, for rows of d elements at every combination of the
// axes; fails where two rows share an element (a stride below the extent of the axes of smaller strides).
inline int extent(Axis *ax, int count, uint64_t d, uint64_t *out) {
    std::sort(ax, ax + count, [](const Axis &x, const Axis &y) { return x.stride < y.stride; });
    uint64_t span = d;
    for (int i = 0; i < count; ++i) {
        if (ax[i].n <= 1) continue;
        if (ax[i].stride < span) return NC_ERROR_INVALID_VALUE;
        if (ax[i].stride > kMostElements / ax[i].n) return NC_ERROR_OVERFLOW;
        span += (ax[i].n - 1) * ax[i].stride;
        if (span > kMostElements) return NC_ERROR_OVERFLOW;
    }
    *out = span;
    return NC_SUCCESS;
}

inline int resolve(const nc_paged_options *opts, Shape *s) {
    if (!opts) return NC_ERROR_INVALID_VALUE;
    s->o = *opts;
    nc_paged_options &o = s->o;
    if (!o.num_seqs || !o.num_q_heads || !o.num_kv_heads || !o.page_size || !o.num_pages || !o.max_pages)
        return NC_ERROR_INVALID_VALUE;
    if (o.head_dim != 16 && o.head_dim != 32 && o.head_dim != 64 && o.head_dim != 128) return NC_ERROR_INVALID_VALUE;
    if (o.element_type != NC_ELEMENT_F16 && o.element_type != NC_ELEMENT_BF16) return NC_ERROR_INVALID_VALUE;
    if (o.num_q_heads % o.num_kv_heads) return NC_ERROR_INVALID_VALUE;
    const uint64_t counts[] = {o.num_seqs, o.num_q_heads, o.page_size, o.num_pages, o.max_pages};
    for (uint64_t n : counts)
        if (n > kMost31) return NC_ERROR_OVERFLOW;
    if (o.page_size * o.num_pages > kMost31 || o.page_size * o.max_pages > kMost31) return NC_ERROR_OVERFLOW;
    if (o.num_q_heads > kMost31 / o.head_dim) return NC_ERROR_OVERFLOW;  // numbers of one request's outputs
    s->group = o.num_q_heads / o.num_kv_heads;
    const uint64_t given[] = {o.table_stride, o.page_stride, o.head_stride, o.token_stride, o.row_stride, o.row_head_stride,
                              o.q_stride, o.q_head_stride, o.o_stride, o.o_head_stride};
    for (uint64_t x : given)
        if (x > kMostElements) return NC_ERROR_OVERFLOW;
    // Workgroups' shares are counted in units, in 32 bits.
    s->heads = o.num_kv_heads * nc_paged_head_parts((uint32_t)s->group);
    const uint64_t keys = nc_paged_step_keys((uint32_t)o.head_dim) * (NC_PAGED_WAVES >> nc_paged_wave_shift((uint32_t)s->group));
    s->seq_units = (o.page_size * o.max_pages + keys - 1) / keys + nc_paged_head_units((uint32_t)o.head_dim);
    if (o.num_seqs * s->heads > kMostUnits || s->seq_units > kMostUnits / (o.num_seqs * s->heads)) return NC_ERROR_OVERFLOW;

    const uint64_t d = o.head_dim;
    o.table_stride = or_packed(o.table_stride, o.max_pages, 1);
    o.token_stride = or_packed(o.token_stride, 1, d);
    // packed values of given inner strides, each at most 2^60: checked before they are multiplied
    if (o.token_stride > kMostElements / o.page_size) return NC_ERROR_OVERFLOW;
    o.head_stride = or_packed(o.head_stride, o.page_size, o.token_stride);
    if (o.head_stride > kMostElements / o.num_kv_heads) return NC_ERROR_OVERFLOW;
    if (!o.page_stride) o.page_stride = std::max(o.num_kv_heads * o.head_stride, o.page_size * o.token_stride);
    o.row_head_stride = or_packed(o.row_head_stride, 1, d);
    if (o.row_head_stride > kMostElements / o.num_kv_heads) return NC_ERROR_OVERFLOW;
    o.row_stride = or_packed(o.row_stride, o.num_kv_heads, o.row_head_stride);
    o.q_head_stride = or_packed(o.q_head_stride, 1, d);
    o.o_head_stride = or_packed(o.o_head_stride, 1, d);
    if (std::max(o.q_head_stride, o.o_head_stride) > kMostElements / o.num_q_heads) return NC_ERROR_OVERFLOW;
    o.q_stride = or_packed(o.q_stride, o.num_q_heads, o.q_head_stride);
    o.o_stride = or_packed(o.o_stride, o.num_q_heads, o.o_head_stride);
    if ((o.page_stride | o.head_stride | o.token_stride) % 8) return NC_ERROR_INVALID_VALUE;

    Axis cache[] = {{o.num_pages, o.page_stride}, {o.num_kv_heads, o.head_stride}, {o.page_size, o.token_stride}};
    Axis table[] = {{o.num_seqs, o.table_stride}};
    Axis q[] = {{o.num_seqs, o.q_stride}, {o.num_q_heads, o.q_head_stride}};
    Axis out[] = {{o.num_seqs, o.o_stride}, {o.num_q_heads, o.o_head_stride}};
    int st = extent(cache, 3, d, &s->cache_len);
    if (!st) st = extent(table, 1, o.max_pages, &s->table_len);
    if (!st) st = extent(q, 2, d, &s->q_len);
    if (!st) st = extent(out, 2, d, &s->o_len);
    if (st) return st;
    // one row's heads; how many rows there are is an argument of the append
    Axis row[] = {{2, o.row_stride}, {o.num_kv_heads, o.row_head_stride}};
    uint64_t unused;
    return extent(row, 2, d, &unused);
}

struct Range {
    uintptr_t lo, hi;
};

inline Range range_of(const void *p, uint64_t elements, uint64_t size) {
    return {reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + elements * size};
}

inline bool overlap(const Range &x, const Range &y) { return x.lo < x.hi && y.lo < y.hi && x.lo < y.hi && y.lo < x.hi; }

// Whether two sets of rows of d elements on the same axes share an element, the second `delta` elements behind the first:
// whether delta + sum i_k stride_k, |i_k| < n_k, comes within d of 0. The axes ascend as extent() leaves them, and
// those below a stride reach less far than it: one of the three multiples about -delta is the only one that can.
inline bool rows_meet(const Axis *ax, int count, int64_t d, int64_t delta) {
    if (count == 0) return delta > -d && delta < d;
    const Axis &x = ax[count - 1];
    if (x.n <= 1) return rows_meet(ax, count - 1, d, delta);
    const int64_t stride = (int64_t)x.stride, most = (int64_t)x.n - 1, near = -(delta / stride);
    for (int64_t i = std::max(near - 1, -most); i <= std::min(near + 1, most); ++i)
        if (rows_meet(ax, count - 1, d, delta + i * stride)) return true;
    return false;
}

inline uintptr_t address(const void *p) { return reinterpret_cast<uintptr_t>(p); }

// The attention's kernel, grid and workspace for a set of options.
struct DecodePlan {
    uint32_t size, odd;  // which of the kernels: by head_dim (0 for 16), and for pages that a 16-key tile may pass the end of
    uint32_t grid, rows, wave_shift, side, many, each_least, long_log2, short_log2, next_least;
    uint64_t piece_ml, piece_o, bytes;  // offsets of the partials, and all of the workspace
    uint64_t score_pitch, row_ml, scores;  // of the scores, where they are kept
};

constexpr uint32_t kCusLog2 = 8;  // MI355X: 256 CUs

// four: a cache in 4 bits; mass: the scores are kept, by kernels of one kind.
inline DecodePlan decode_plan(const Shape &s, bool o_vec, bool four = false, bool mass = false) {
    const nc_paged_options &o = s.o;
    DecodePlan p;
    // A 16-key tile lies in one page, and a page's byte offsets fit 32 bits.
    // (4 bits: so do the whole pool's values.)
    const bool uniform = o.page_size % 16 == 0 && (four ? s.cache_len <= 0xffffffffull : o.page_stride < (1ull << 31) && o.page_size * o.token_stride < (1ull << 30));
    const uint32_t d = o.head_dim == 16 ? 0 : o.head_dim == 32 ? 1 : o.head_dim == 64 ? 2 : 3;
    // Workgroups for long heads: one per CU for heads of 64 and 128, whose loads are wide. Two for small heads, and on pages of
    // any size where waves share their keys and have half as much under way. 4 requests of 20000 over 4 key heads, 20 query
    // heads each, one and two per CU:
    //   pages of 24   heads of 64  39.2  31.1 us    heads of 128  59.6  54.3
    //   pages of 16   heads of 64  32.9  30.9       heads of 128  54.2  55.9   (96 of 4000 over 8 of 64: 167  175)
    const bool two = o.head_dim <= 32 || (!uniform && s.group > 16);
    const uint32_t head_units = four ? nc_paged4_head_units((uint32_t)o.head_dim) : nc_paged_head_units((uint32_t)o.head_dim);
    // 4 bits: two as well, whose loads hide each other's steps, but for a few heads, whose pieces they double. One and two per CU:
    //   96 requests of 4000 over 8 heads of 64, 8 query heads each   82.6  66.6 us     16 of 4000 over 8 of 128   22.1  21.7
    //   2 of 20000 over 8 of 64, 8 query heads each                  15.6  18.2        one of 30000 over 8 of 128  17.9  18.7
    p.long_log2 = kCusLog2 + (two || (four && o.num_seqs * s.heads > 16) ? 1 : 0);
    // Short heads: as many as are resident. (Heads of 64 and 128 with twice as many: 512 requests of 100 over 8 heads of 128
    // 48.6 -> 50.0 us.)
    p.short_log2 = kCusLog2 + (o.head_dim <= 32 ? 2 : 1);
    // Where a token's heads are next to each other and its neighbour's rows are not, two or four waves take neighbouring heads
    // of the same keys rather than different keys of one head, if their pieces stay small. Small heads share a 128-byte line;
    // wide ones gain by their order in memory, unless there are many. Each head for itself and neighbouring ones:
    //   100 requests of 4000 over 4 heads of 16, pages of 1             67.6  36.8 us
    //   200 of up to 1000 over 8 heads of 16                            18.7  13.3
    //   16 of 6000 over 2 heads of 16, 16 query heads each              10.8  13.4 (not taken: large pieces)
    //   one of 120001 over 8 heads of 64                                59.1  54.5
    //   8 of 4000 over 8 heads of 128                                   31.9  30.5
    //   30 of up to 6000 over 2 heads of 128                            12.9  14.2 (not taken: two heads)
    //   160 of 3000 over 8 heads of 128                                331   338   (not taken: many; but 100 of up to 2000
    //                                               over 32 heads would be 105 and 87, 200 of up to 4000 over 8 of 64 57 and 46)
    // Short requests are faster over all waves, so the kernel looks at the lengths (NC_PAGED_NEXT_TOKENS; 0.1 to 0.3 us where it
    // finds them short); where the table has no room for a long one, it need not.
    uint32_t side = 0;
    p.next_least = 0;
    if ((!mass || four) && (o.head_stride < o.token_stride || o.page_size == 1) && o.max_pages * o.page_size > NC_PAGED_NEXT_TOKENS) {
        const uint64_t numbers = s.group * o.head_dim;  // of one head's piece
        // 4 bits: rows are a quarter as long, and neighbouring heads' share lines up to heads of 128. Each head for itself, two, four:
        //   one request of 120001 over 8 heads of 64                 46.0  31.2  32.0 us
        //   16 of 2000 over 8 heads of 128                           21.9  18.9
        //   100 of 600 over 32 heads of 64                           121   70    62.6
        //   32 of 4000 over 4 of 64, 8 query heads each, pages of 1  32.9        26.4
        //   4 of 5000 over 8 of 128, pages of 24                     19.1  21.3       (not taken: addresses by key, and few heads)
        //   16 of 4000 over 8 of 128, pages of 7                     36.2  26.7
        //   64 of 4000 over 8 of 128, pages of 24                   102.3  80.8       (8 of 2000: 16.0  15.7)
        //   16 of 4000 over 8 of 128, pages of 1                     40.2  29.8  33.5
        //   the same, 8 query heads each, ragged                     18.5  22.8  33.0
        if (four) {
            const bool narrow = o.head_dim <= 64, pair = narrow || uniform || o.num_seqs * s.heads > 32;
            // (wide: only where the lengths say that there is much to read, NC_PAGED4_WIDE_UNITS)
            const bool wide = s.group > 4 && !(narrow && o.page_size == 1);  // pieces
            side = s.group > 8 ? 0 : o.num_kv_heads % 4 == 0 && narrow && !wide ? 2 : o.num_kv_heads % 2 == 0 && pair ? 1 : 0;
            if (wide) p.next_least = NC_PAGED4_WIDE_UNITS;
        }
        else if (o.head_dim <= 32)
            side = o.num_kv_heads % 4 == 0 && numbers <= 64 ? 2 : o.num_kv_heads % 2 == 0 && numbers <= 128 ? 1 : 0;
        else
            side = o.num_kv_heads % 4 == 0 && s.group <= 4 && o.num_seqs * s.heads <= 2u << p.short_log2;
    }
    p.wave_shift = nc_paged_wave_shift((uint32_t)s.group);
    p.side = side;
    p.rows = (uint32_t)std::min<uint64_t>(s.group, 64);
    const uint64_t step = four ? NC_PAGED4_STEP_KEYS : nc_paged_step_keys((uint32_t)o.head_dim);
    // A piece is written and read once more: at most a quarter of what its run reads of the cache. (Neighbouring heads' are at
    // most 16 rows, and no more than a block's reads.)
    p.each_least = (uint32_t)std::max<uint64_t>(1, 8 * p.rows / (step * (NC_PAGED_WAVES >> p.wave_shift)));
    // Units there may be, in both ways of taking the heads.
    auto units = [&](uint64_t heads, uint32_t shift) {
        const uint64_t keys = step * (NC_PAGED_WAVES >> shift);
        return o.num_seqs * heads * ((o.page_size * o.max_pages + keys - 1) / keys + head_units);
    };
    const uint64_t most = std::max(units(s.heads, p.wave_shift), side ? units(s.heads >> side, side) : 0);
    p.grid = (uint32_t)std::min<uint64_t>(most, 1u << p.short_log2);
    const uint64_t rows = std::max<uint64_t>(p.rows, side ? s.group << side : 0);
    // More heads than workgroups: where a workgroup has several short ones, its waves take one each. Without and with:
    //   200 requests of 60, 32 heads of 64, pages of 24   42.7  26.7 us
    //   256 of 50, 8 heads of 128                         15.8  13.2
    //   128 of 120, 8 heads of 128, two a workgroup       14.1  14.1
    // That code makes a call up to 0.1 us longer, so it has kernels of its own.
    p.many = (!mass || four) && s.group <= 16 && o_vec && o.num_seqs * s.heads > 1u << p.short_log2;
    p.size = d;
    p.odd = uniform ? 0 : 1;
    p.piece_ml = NC_PAGED_ROUNDS * 2 * NC_PAGED_MAX_WGS * 4;
    p.piece_o = p.piece_ml + p.grid * 2 * rows * 2 * 4;
    p.bytes = p.piece_o + p.grid * 2 * rows * o.head_dim * 4;
    p.score_pitch = p.row_ml = p.scores = 0;
    if (mass) {  // a row of scores holds whole 16-key tiles
        p.score_pitch = (o.max_pages * o.page_size + 15) / 16 * 16;
        p.row_ml = p.bytes = (p.bytes + 15) / 16 * 16;
        p.scores = p.bytes = (p.bytes + o.num_seqs * o.num_q_heads * 8 + 15) / 16 * 16;
        p.bytes += o.num_seqs * o.num_q_heads * p.score_pitch * 4;
    }
    return p;
}

// The attention's tensors beside the cache.
struct DecodeTensors {
    const uint16_t *q;
    uint64_t q_len;
    const int32_t *block_table;
    uint64_t table_len;
    const int32_t *seq_lens;
    uint64_t lens_len;
    float *o;
    uint64_t o_len;
    void *workspace;
    uint64_t workspace_bytes;
};

inline bool o_is_vec(const Shape &s, const float *o) { return address(o) % 16 == 0 && (s.o.o_stride | s.o.o_head_stride) % 4 == 0; }

// Whether they are there, long enough and aligned.
inline int check_decode(const Shape &s, const DecodePlan &plan, const DecodeTensors &t) {
    if (!t.q || !t.block_table || !t.seq_lens || !t.o || !t.workspace) return NC_ERROR_INVALID_VALUE;
    if (t.q_len < s.q_len || t.table_len < s.table_len || t.lens_len < s.o.num_seqs || t.o_len < s.o_len || t.workspace_bytes < plan.bytes)
        return NC_ERROR_INVALID_VALUE;
    if (address(t.workspace) % 16 || address(t.q) % 2 || (address(t.block_table) | address(t.seq_lens) | address(t.o)) % 4)
        return NC_ERROR_INVALID_VALUE;
    return NC_SUCCESS;
}

// Whether O or the workspace overlaps another of these, or one of `count` more ranges.
inline bool decode_overlaps(const Shape &s, const DecodePlan &plan, const DecodeTensors &t, const Range *more, int count) {
    const Range outs[] = {range_of(t.o, s.o_len, 4), range_of(t.workspace, plan.bytes, 1)};
    const Range ins[] = {range_of(t.q, s.q_len, 2), range_of(t.block_table, s.table_len, 4), range_of(t.seq_lens, s.o.num_seqs, 4)};
    bool bad = overlap(outs[0], outs[1]);
    for (const Range &x : outs) {
        for (const Range &y : ins) bad = bad || overlap(x, y);
        for (int i = 0; i < count; ++i) bad = bad || overlap(x, more[i]);
    }
    return bad;
}

inline void decode_args(const Shape &s, const DecodePlan &plan, const DecodeTensors &t, const void *k, const void *v, nc_paged_decode_args *args) {
    nc_paged_decode_args &a = *args;
    const nc_paged_options &op = s.o;
    a.q = t.q;
    a.k = static_cast<const uint16_t *>(k);
    a.v = static_cast<const uint16_t *>(v);
    a.table = t.block_table;
    a.seq_lens = t.seq_lens;
    a.o = t.o;
    a.counters = static_cast<uint32_t *>(t.workspace);
    a.part_ml = reinterpret_cast<float *>(static_cast<char *>(t.workspace) + plan.piece_ml);
    a.part_o = reinterpret_cast<float *>(static_cast<char *>(t.workspace) + plan.piece_o);
    a.rows = plan.rows;
    a.wave_shift = plan.wave_shift;
    a.side = plan.side;
    a.many = plan.many;
    a.long_log2 = plan.long_log2;
    a.short_log2 = plan.short_log2;
    a.each_least = plan.each_least;
    a.heads = nc_paged_make_div((uint32_t)s.heads);
    a.group_inverse = (uint32_t)(65536 / s.group + 1);
    a.head_parts = nc_paged_head_parts((uint32_t)s.group);
    a.q_vec = address(t.q) % 16 == 0 && (op.q_stride | op.q_head_stride) % 8 == 0;
    a.o_vec = o_is_vec(s, t.o);
    a.table_stride = op.table_stride;
    a.page_stride = op.page_stride;
    a.head_stride = op.head_stride;
    a.token_stride = op.token_stride;
    a.q_stride = op.q_stride;
    a.q_head_stride = op.q_head_stride;
    a.o_stride = op.o_stride;
    a.o_head_stride = op.o_head_stride;
    a.num_seqs = (uint32_t)op.num_seqs;
    a.num_q_heads = (uint32_t)op.num_q_heads;
    a.num_kv_heads = (uint32_t)op.num_kv_heads;
    a.group = (uint32_t)s.group;
    a.num_pages = (uint32_t)op.num_pages;
    a.max_tokens = (uint32_t)(op.max_pages * op.page_size);
    a.scale = op.scale;
    a.ps = nc_paged_make_div((uint32_t)op.page_size);
}

inline int launch_kernel(nc_module module, uint32_t slot, const char *name, uint32_t grid, uint32_t grid_y, uint32_t threads, void *args, nc_stream stream) {
    nc_function fn = nullptr;
    int st = nc_internal_module_kept_function(module, slot, name, &fn);
    if (st) return st;
    nc_launch_config cfg;
    std::memset(&cfg, 0, sizeof cfg);
    cfg.grid[0] = grid;
    cfg.grid[1] = grid_y;
    cfg.grid[2] = 1;
    cfg.block[0] = threads;
    cfg.block[1] = cfg.block[2] = 1;
    cfg.stream = stream;
    void *params[] = {args};
    return nc_function_launch(fn, &cfg, params);
}

}  // namespace nc_paged

#endif
