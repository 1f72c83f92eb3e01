// paged.cpp — host side of the paged key-value cache (include/notcute_paged.h): validation, the choice of
// kernel and grid, launches. Nothing here allocates or synchronises.

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "notcute_paged.h"
#include "paged_args.h"

extern "C" int nc_internal_fail(int status, const char *what);
// hip_api.cpp: a function of the module, looked up once and kept under `slot` (below NC_PAGED_KERNELS).
extern "C" int nc_internal_module_kept_function(nc_module module, uint32_t slot, const char *name, nc_function *out);

namespace {

constexpr uint64_t kMost31 = 0x7fffffffull;
constexpr uint64_t kMostUnits = 1ull << 30;
constexpr uint64_t kMostElements = 1ull << 60;

// The options with every stride resolved.
struct Shape {
    nc_paged_options o;
    uint64_t group, cache_len, table_len, q_len, o_len;
    uint64_t heads, seq_units;  // the attention's: key heads (parts of them), and most units of a head
};

uint64_t or_packed(uint64_t stride, uint64_t count, uint64_t inner) { return stride ? stride : count * inner; }

struct Axis {
    uint64_t n, stride;
};

// Elements from a tensor's first to behind its last, for rows of d elements at every combination of the
// axes; fails where two rows share an element (a stride below the extent of the axes of smaller strides).
int extent(Axis *ax, int count, uint64_t d, uint64_t *out) {
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

int resolve(const nc_paged_options *opts, Shape *s) {
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

Range range_of(const void *p, uint64_t elements, uint64_t size) {
    return {reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + elements * size};
}

bool overlap(const Range &x, const Range &y) { return x.lo < x.hi && y.lo < y.hi && x.lo < y.hi && y.lo < x.hi; }

// Whether two sets of rows of d elements on the same axes share an element, the second `delta` elements behind the first:
// whether delta + sum i_k stride_k, |i_k| < n_k, comes within d of 0. The axes ascend as extent() leaves them, and
// those below a stride reach less far than it: one of the three multiples about -delta is the only one that can.
bool rows_meet(const Axis *ax, int count, int64_t d, int64_t delta) {
    if (count == 0) return delta > -d && delta < d;
    const Axis &x = ax[count - 1];
    if (x.n <= 1) return rows_meet(ax, count - 1, d, delta);
    const int64_t stride = (int64_t)x.stride, most = (int64_t)x.n - 1, near = -(delta / stride);
    for (int64_t i = std::max(near - 1, -most); i <= std::min(near + 1, most); ++i)
        if (rows_meet(ax, count - 1, d, delta + i * stride)) return true;
    return false;
}

uintptr_t address(const void *p) { return reinterpret_cast<uintptr_t>(p); }

// Every kernel of paged.hip by its place here, under which the module keeps its function.
#define NC_DECODE_NAMES(D)                                                                \
    "nc_paged_decode_d" #D, "nc_paged_decode_d" #D "_bf16", "nc_paged_decode_d" #D "_odd", \
        "nc_paged_decode_d" #D "_odd_bf16", "nc_paged_decode_d" #D "_many",               \
        "nc_paged_decode_d" #D "_many_bf16", "nc_paged_decode_d" #D "_many_odd",          \
        "nc_paged_decode_d" #D "_many_odd_bf16", "nc_paged_decode_d" #D "_next",          \
        "nc_paged_decode_d" #D "_next_bf16", "nc_paged_decode_d" #D "_next_odd", "nc_paged_decode_d" #D "_next_odd_bf16"
const char *const kKernels[] = {
    "nc_paged_build",
    "nc_paged_append_rows",
    "nc_paged_append_rows_unaligned",
    "nc_paged_append_rows_d16",
    "nc_paged_append_rows_d16_unaligned",
    NC_DECODE_NAMES(16),
    NC_DECODE_NAMES(32),
    NC_DECODE_NAMES(64),
    NC_DECODE_NAMES(128),
};
enum : uint32_t { kBuild, kAppend, kAppendD16 = kAppend + 2, kDecode = kAppend + 4 };

int launch(nc_module module, uint32_t kernel, uint32_t grid, uint32_t threads, void *args, nc_stream stream) {
    nc_function fn = nullptr;
    int st = nc_internal_module_kept_function(module, kernel, kKernels[kernel], &fn);
    if (st) return st;
    nc_launch_config cfg;
    std::memset(&cfg, 0, sizeof cfg);
    cfg.grid[0] = grid;
    cfg.grid[1] = cfg.grid[2] = 1;
    cfg.block[0] = threads;
    cfg.block[1] = cfg.block[2] = 1;
    cfg.stream = stream;
    void *params[] = {args};
    return nc_function_launch(fn, &cfg, params);
}

// The attention's kernel, grid and workspace for a set of options.
struct DecodePlan {
    uint32_t kernel, grid, rows, wave_shift, side, many, each_least, long_log2, short_log2;
    uint64_t piece_ml, piece_o, bytes;  // offsets of the partials, and all of the workspace
};

constexpr uint32_t kCusLog2 = 8;  // MI355X: 256 CUs

DecodePlan decode_plan(const Shape &s, bool o_vec) {
    const nc_paged_options &o = s.o;
    DecodePlan p;
    // A 16-key tile lies in one page, and a page's byte offsets fit 32 bits.
    const bool uniform = o.page_size % 16 == 0 && o.page_stride < (1ull << 31) && o.page_size * o.token_stride < (1ull << 30);
    const uint32_t d = o.head_dim == 16 ? 0 : o.head_dim == 32 ? 1 : o.head_dim == 64 ? 2 : 3;
    // Workgroups for long heads: one per CU for heads of 64 and 128, whose loads are wide. Two for small heads, and on pages of
    // any size where waves share their keys and have half as much under way. 4 requests of 20000 over 4 key heads, 20 query
    // heads each, one and two per CU:
    //   pages of 24   heads of 64  39.2  31.1 us    heads of 128  59.6  54.3
    //   pages of 16   heads of 64  32.9  30.9       heads of 128  54.2  55.9   (96 of 4000 over 8 of 64: 167  175)
    const bool two = o.head_dim <= 32 || (!uniform && s.group > 16);
    p.long_log2 = kCusLog2 + (two ? 1 : 0);
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
    if ((o.head_stride < o.token_stride || o.page_size == 1) && o.max_pages * o.page_size > NC_PAGED_NEXT_TOKENS) {
        const uint64_t numbers = s.group * o.head_dim;  // of one head's piece
        if (o.head_dim <= 32)
            side = o.num_kv_heads % 4 == 0 && numbers <= 64 ? 2 : o.num_kv_heads % 2 == 0 && numbers <= 128 ? 1 : 0;
        else
            side = o.num_kv_heads % 4 == 0 && s.group <= 4 && o.num_seqs * s.heads <= 2u << p.short_log2;
    }
    p.wave_shift = nc_paged_wave_shift((uint32_t)s.group);
    p.side = side;
    p.rows = (uint32_t)std::min<uint64_t>(s.group, 64);
    const uint64_t step = nc_paged_step_keys((uint32_t)o.head_dim);
    // A piece is written and read once more: at most a quarter of what its run reads of the cache. (Neighbouring heads' are at
    // most 16 rows, and no more than a block's reads.)
    p.each_least = (uint32_t)std::max<uint64_t>(1, 8 * p.rows / (step * (NC_PAGED_WAVES >> p.wave_shift)));
    // Units there may be, in both ways of taking the heads.
    auto units = [&](uint64_t heads, uint32_t shift) {
        const uint64_t keys = step * (NC_PAGED_WAVES >> shift);
        return o.num_seqs * heads * ((o.page_size * o.max_pages + keys - 1) / keys + nc_paged_head_units((uint32_t)o.head_dim));
    };
    const uint64_t most = std::max(units(s.heads, p.wave_shift), side ? units(s.heads >> side, side) : 0);
    p.grid = (uint32_t)std::min<uint64_t>(most, 1u << p.short_log2);
    const uint64_t rows = std::max<uint64_t>(p.rows, side ? s.group << side : 0);
    // More heads than workgroups: where a workgroup has several short ones, its waves take one each. Without and with:
    //   200 requests of 60, 32 heads of 64, pages of 24   42.7  26.7 us
    //   256 of 50, 8 heads of 128                         15.8  13.2
    //   128 of 120, 8 heads of 128, two a workgroup       14.1  14.1
    // That code makes a call up to 0.1 us longer, so it has kernels of its own.
    p.many = s.group <= 16 && o_vec && o.num_seqs * s.heads > 1u << p.short_log2;
    p.kernel = kDecode + 12 * d + (side ? 8 : p.many ? 4 : 0) + (uniform ? 0 : 2) + (o.element_type == NC_ELEMENT_BF16 ? 1 : 0);
    p.piece_ml = NC_PAGED_ROUNDS * 2 * NC_PAGED_MAX_WGS * 4;
    p.piece_o = p.piece_ml + p.grid * 2 * rows * 2 * 4;
    p.bytes = p.piece_o + p.grid * 2 * rows * o.head_dim * 4;
    return p;
}

static_assert(sizeof kKernels / sizeof kKernels[0] == NC_PAGED_KERNELS, "one place per kernel");

}  // namespace

extern "C" {

void nc_paged_options_init(nc_paged_options *opts) {
    if (!opts) return;
    std::memset(opts, 0, sizeof *opts);
    opts->num_seqs = opts->num_q_heads = opts->num_kv_heads = opts->max_pages = 1;
}

int nc_paged_validate(const nc_paged_options *opts) {
    Shape s;
    return resolve(opts, &s);
}

uint64_t nc_paged_workspace_bytes(const nc_paged_options *opts) {
    Shape s;
    return resolve(opts, &s) ? 0 : decode_plan(s, true).bytes;
}

int nc_paged_build(nc_module module, const nc_paged_build_buffers *buffers, const nc_paged_options *opts,
                   nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged_build_buffers &t = *buffers;
    Shape s;
    int st = resolve(opts, &s);
    if (st) return st;
    const nc_paged_options &o = s.o;
    if (!module || !t.cached_lens || !t.new_lens || !t.cursor || !t.block_table || !t.seq_lens || !t.row_offsets || !t.counts ||
        (!t.free_pages && t.free_len) || (!t.slots && t.slots_len))
        return NC_ERROR_INVALID_VALUE;
    if (t.cached_len < o.num_seqs || t.new_len < o.num_seqs || t.seq_len < o.num_seqs || t.offsets_len < o.num_seqs + 1 ||
        t.table_len < s.table_len || t.cursor_len < 1 || t.counts_len < 4)
        return NC_ERROR_INVALID_VALUE;
    if (t.slots_len > kMost31 || t.free_len > kMost31) return NC_ERROR_OVERFLOW;
    if ((address(t.cached_lens) | address(t.new_lens) | address(t.free_pages) | address(t.cursor) | address(t.block_table) |
         address(t.seq_lens) | address(t.row_offsets) | address(t.slots) | address(t.counts)) % 4)
        return NC_ERROR_INVALID_VALUE;

    // Outputs first; a pair may be one and the same buffer only where the header says so.
    const Range rg[] = {range_of(t.seq_lens, o.num_seqs, 4),    range_of(t.counts, 4, 4),
                        range_of(t.block_table, s.table_len, 4), range_of(t.row_offsets, o.num_seqs + 1, 4),
                        range_of(t.slots, t.slots_len, 4),         range_of(t.cached_lens, o.num_seqs, 4),
                        range_of(t.cursor, 1, 4),                range_of(t.new_lens, o.num_seqs, 4),
                        range_of(t.free_pages, t.free_len, 4)};
    const bool same_lens = t.seq_lens == t.cached_lens, same_cursor = t.counts == t.cursor;
    for (int i = 0; i < 5; ++i)
        for (int j = i + 1; j < 9; ++j) {
            if ((i == 0 && j == 5 && same_lens) || (i == 1 && j == 6 && same_cursor)) continue;
            if (overlap(rg[i], rg[j]))
                return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_build: an output overlaps another buffer");
        }

    nc_paged_build_args a;
    std::memset(&a, 0, sizeof a);
    a.cached = t.cached_lens;
    a.fresh = t.new_lens;
    a.free_pages = t.free_pages;
    a.cursor = t.cursor;
    a.table = t.block_table;
    a.seq_lens = t.seq_lens;
    a.offsets = t.row_offsets;
    a.slots = t.slots;
    a.counts = t.counts;
    a.table_stride = o.table_stride;
    a.num_seqs = (uint32_t)o.num_seqs;
    a.width = (uint32_t)o.max_pages;
    a.num_pages = (uint32_t)o.num_pages;
    a.free_len = (uint32_t)t.free_len;
    a.places = (uint32_t)t.slots_len;
    a.ps = nc_paged_make_div((uint32_t)o.page_size);
    const uint32_t threads = o.num_seqs <= 64 ? 64 : o.num_seqs <= 256 ? 256 : 1024;
    // One workgroup where its threads write a slot each, or a request's thread its few. Else a slot a thread, or two where a
    // workgroup needs several rounds to scan the requests. This rule, twice as many a thread, and all in one workgroup:
    //   3 requests of up to 946 rows, 1400 together   4.0   4.5   17 us
    //   256 of up to 4096, 121000 together            5.3   5.8  337
    //   2000 of up to 2000, 530000 together          11.4  12.8  454
    const uint64_t chunk = threads * (o.num_seqs > 1024 ? 2 : 1);
    const uint64_t single = std::max<uint64_t>(threads, std::min<uint64_t>(4096, 8 * o.num_seqs));
    const uint64_t wgs = t.slots_len <= single ? 1 : std::min<uint64_t>((t.slots_len + chunk - 1) / chunk, 1024);
    a.chunk_rows = (uint32_t)((t.slots_len + wgs - 1) / wgs);
    // no more pages than this are taken
    const uint64_t pages = std::min<uint64_t>(t.free_len, t.slots_len / o.page_size + o.num_seqs);
    a.chunk_pages = (uint32_t)((pages + wgs - 1) / wgs);
    a.parts = NC_PAGED_PART_PAGES | NC_PAGED_PART_LENS;
    // In place, several workgroups read what one of them would write: the lengths wait for a second launch.
    const bool later = wgs > 1 && (same_lens || same_cursor);
    if (later) a.parts = NC_PAGED_PART_PAGES;
    st = launch(module, kBuild, (uint32_t)wgs, threads, &a, stream);
    if (st || !later) return st;
    a.parts = NC_PAGED_PART_LENS;
    return launch(module, kBuild, 1, threads, &a, stream);
}

int nc_paged_append(nc_module module, const nc_paged_append_buffers *buffers, const nc_paged_options *opts,
                    nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged_append_buffers &t = *buffers;
    Shape s;
    int st = resolve(opts, &s);
    if (st) return st;
    const nc_paged_options &o = s.o;
    if (!module || !t.k_cache || !t.v_cache || t.k_len < s.cache_len || t.v_len < s.cache_len) return NC_ERROR_INVALID_VALUE;
    if ((address(t.k_cache) | address(t.v_cache)) % 16) return NC_ERROR_INVALID_VALUE;
    const Range caches[] = {range_of(t.k_cache, s.cache_len, 2), range_of(t.v_cache, s.cache_len, 2)};
    // K and V may be interleaved, but no row of one may be part of a row of the other.
    Axis cache[] = {{o.num_pages, o.page_stride}, {o.num_kv_heads, o.head_stride}, {o.page_size, o.token_stride}};
    uint64_t unused;
    st = extent(cache, 3, o.head_dim, &unused);
    if (st) return st;
    const int64_t apart = (int64_t)(address(t.v_cache) - address(t.k_cache)) / 2;
    if (overlap(caches[0], caches[1]) && rows_meet(cache, 3, (int64_t)o.head_dim, apart))
        return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_append: rows of K and V share memory");
    if (t.num_rows == 0) return NC_SUCCESS;
    if (t.num_rows > kMost31) return NC_ERROR_OVERFLOW;
    Axis row[] = {{t.num_rows, o.row_stride}, {o.num_kv_heads, o.row_head_stride}};
    uint64_t rows_len = 0;
    st = extent(row, 2, o.head_dim, &rows_len);
    if (st) return st;
    if (!t.k_rows || !t.v_rows || !t.slots || t.k_rows_len < rows_len || t.v_rows_len < rows_len || t.slots_len < t.num_rows)
        return NC_ERROR_INVALID_VALUE;
    if ((address(t.k_rows) | address(t.v_rows)) % 2 || address(t.slots) % 4) return NC_ERROR_INVALID_VALUE;
    const Range ins[] = {range_of(t.k_rows, rows_len, 2), range_of(t.v_rows, rows_len, 2), range_of(t.slots, t.num_rows, 4)};
    for (const Range &x : caches)
        for (const Range &y : ins)
            if (overlap(x, y)) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_append: the rows overlap the cache");

    nc_paged_append_args a;
    std::memset(&a, 0, sizeof a);
    a.k_rows = t.k_rows;
    a.v_rows = t.v_rows;
    a.slots = t.slots;
    a.k = t.k_cache;
    a.v = t.v_cache;
    a.row_stride = o.row_stride;
    a.row_head_stride = o.row_head_stride;
    a.page_stride = o.page_stride;
    a.head_stride = o.head_stride;
    a.token_stride = o.token_stride;
    a.num_rows = t.num_rows;
    a.num_slots = (uint32_t)(o.num_pages * o.page_size);
    a.ps = nc_paged_make_div((uint32_t)o.page_size);
    const uint64_t chunks = o.num_kv_heads * (o.head_dim / 8);
    if (chunks > kMost31 / 2) return NC_ERROR_OVERFLOW;
    a.chunks = nc_paged_make_div((uint32_t)chunks);
    a.chunk_shift = o.head_dim == 16 ? 1 : o.head_dim == 32 ? 2 : o.head_dim == 64 ? 3 : 4;
    // a chunk a thread, and no more than 2^23 workgroups
    a.wg_rows = (uint32_t)std::max<uint64_t>(std::max<uint64_t>(1, 256 / chunks), (t.num_rows + (1u << 23) - 1) >> 23);
    if (a.wg_rows * chunks > kMost31) return NC_ERROR_OVERFLOW;
    const bool vec = (address(t.k_rows) | address(t.v_rows)) % 16 == 0 && (o.row_stride | o.row_head_stride) % 8 == 0;
    return launch(module, (o.head_dim == 16 ? kAppendD16 : kAppend) + (vec ? 0 : 1),
                  (uint32_t)((t.num_rows + a.wg_rows - 1) / a.wg_rows), 256, &a, stream);
}

int nc_paged_decode(nc_module module, const nc_paged_decode_buffers *buffers, const nc_paged_options *opts,
                    nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged_decode_buffers &t = *buffers;
    Shape s;
    int st = resolve(opts, &s);
    if (st) return st;
    const nc_paged_options &op = s.o;
    const bool o_vec = address(t.o) % 16 == 0 && (op.o_stride | op.o_head_stride) % 4 == 0;
    const DecodePlan plan = decode_plan(s, o_vec);
    const uint64_t need = plan.bytes;
    if (!module || !t.q || !t.k_cache || !t.v_cache || !t.block_table || !t.seq_lens || !t.o || !t.workspace)
        return NC_ERROR_INVALID_VALUE;
    if (t.q_len < s.q_len || t.k_len < s.cache_len || t.v_len < s.cache_len || t.table_len < s.table_len ||
        t.lens_len < op.num_seqs || t.o_len < s.o_len || t.workspace_bytes < need)
        return NC_ERROR_INVALID_VALUE;
    if ((address(t.k_cache) | address(t.v_cache) | address(t.workspace)) % 16 || address(t.q) % 2 ||
        (address(t.block_table) | address(t.seq_lens) | address(t.o)) % 4)
        return NC_ERROR_INVALID_VALUE;
    const Range outs[] = {range_of(t.o, s.o_len, 4), range_of(t.workspace, need, 1)};
    const Range ins[] = {range_of(t.q, s.q_len, 2), range_of(t.k_cache, s.cache_len, 2), range_of(t.v_cache, s.cache_len, 2),
                         range_of(t.block_table, s.table_len, 4), range_of(t.seq_lens, op.num_seqs, 4)};
    bool bad = overlap(outs[0], outs[1]);
    for (const Range &x : outs)
        for (const Range &y : ins) bad = bad || overlap(x, y);
    if (bad) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_decode: O or the workspace overlaps another buffer");

    nc_paged_decode_args a;
    std::memset(&a, 0, sizeof a);
    a.q = t.q;
    a.k = t.k_cache;
    a.v = t.v_cache;
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
    a.o_vec = o_vec;
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
    return launch(module, plan.kernel, plan.grid, 64 * NC_PAGED_WAVES, &a, stream);
}

}  // extern "C"
