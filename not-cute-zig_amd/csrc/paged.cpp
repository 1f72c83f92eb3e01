// paged.cpp — host side of the paged key-value cache (include/notcute_paged.h): validation, the choice of
// kernel and grid, launches. Nothing here allocates or synchronises.

#include "paged_host.h"

using namespace nc_paged;

namespace {

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
    return launch_kernel(module, kernel, kKernels[kernel], grid, 1, threads, args, stream);
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
    const DecodeTensors x = {t.q, t.q_len, t.block_table, t.table_len, t.seq_lens, t.lens_len, t.o, t.o_len, t.workspace, t.workspace_bytes};
    const DecodePlan plan = decode_plan(s, o_is_vec(s, t.o));
    if (!module || !t.k_cache || !t.v_cache || t.k_len < s.cache_len || t.v_len < s.cache_len) return NC_ERROR_INVALID_VALUE;
    if ((address(t.k_cache) | address(t.v_cache)) % 16) return NC_ERROR_INVALID_VALUE;
    st = check_decode(s, plan, x);
    if (st) return st;
    const Range caches[] = {range_of(t.k_cache, s.cache_len, 2), range_of(t.v_cache, s.cache_len, 2)};
    if (decode_overlaps(s, plan, x, caches, 2))
        return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_decode: O or the workspace overlaps another buffer");

    nc_paged_decode_args a;
    std::memset(&a, 0, sizeof a);
    decode_args(s, plan, x, t.k_cache, t.v_cache, &a);
    const uint32_t kernel = kDecode + 12 * plan.size + (plan.side ? 8 : plan.many ? 4 : 0) + 2 * plan.odd + (s.o.element_type == NC_ELEMENT_BF16 ? 1 : 0);
    return launch(module, kernel, plan.grid, 64 * NC_PAGED_WAVES, &a, stream);
}

}  // extern "C"
