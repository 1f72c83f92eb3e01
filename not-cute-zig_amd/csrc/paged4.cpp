// paged4.cpp — host side of the smaller paged cache (include/notcute_paged4.h): validation, the choice of kernel and grid,
// launches. Nothing here allocates or synchronises.

#include "notcute_paged4.h"
#include "paged4_args.h"
#include "paged_host.h"

using namespace nc_paged;

// Looks at other chunks' flags before an eviction's move gives up waiting: some tenth of a second's. Tests lower it.
extern "C" {
uint32_t nc_internal_evict_tries = 1u << 16;
}

namespace {

// Every kernel of paged4.hip by its place here, under which the module keeps its function.
#define NC_DECODE4_NAMES(D, T) \
    "nc_paged4_decode_d" #D T, "nc_paged4_decode_d" #D T "_odd", "nc_paged4_mass4_d" #D T, "nc_paged4_mass4_d" #D T "_odd"
#define NC_DECODE4_ALL(D) NC_DECODE4_NAMES(D, ""), NC_DECODE4_NAMES(D, "_by2"), NC_DECODE4_NAMES(D, "_by4")
#define NC_MASS_NAMES(D) \
    "nc_paged4_mass_d" #D, "nc_paged4_mass_d" #D "_bf16", "nc_paged4_mass_d" #D "_odd", "nc_paged4_mass_d" #D "_odd_bf16"
const char *const kKernels[] = {
    "nc_paged4_append", "nc_paged4_read", "nc_paged4_weights", "nc_paged4_select", "nc_paged4_select_short", "nc_paged4_part_first",
    "nc_paged4_part_second", "nc_paged4_part_third", "nc_paged4_part_list", "nc_paged4_move",
    NC_DECODE4_ALL(32), NC_DECODE4_ALL(64), NC_DECODE4_ALL(128), NC_MASS_NAMES(16), NC_MASS_NAMES(32),
    NC_MASS_NAMES(64),  NC_MASS_NAMES(128),
};
enum : uint32_t { kAppend, kRead, kWeights, kSelect, kSelectShort, kPartFirst, kMove = kPartFirst + 4, kDecode4, kMass = kDecode4 + 3 * 12 };
static_assert(sizeof kKernels / sizeof kKernels[0] == NC_PAGED4_KERNELS, "one place per kernel");

int launch(nc_module module, uint32_t kernel, uint32_t grid, uint32_t grid_y, uint32_t threads, void *args, nc_stream stream) {
    return launch_kernel(module, NC_PAGED_KERNELS + kernel, kKernels[kernel], grid, grid_y, threads, args, stream);
}

// Values of a pool in 4 bits: the kernels count 32 at a time, in 32 bits, of which all ones stand for no place.
constexpr uint64_t kMostValues = (1ull << 37) - 32;

int resolve4(const nc_paged_options *opts, Shape *s) {
    int st = resolve(opts, s);
    if (st) return st;
    if (s->o.head_dim < 32 || (s->o.page_stride | s->o.head_stride | s->o.token_stride) % 32) return NC_ERROR_INVALID_VALUE;
    return s->cache_len > kMostValues ? NC_ERROR_OVERFLOW : NC_SUCCESS;
}

int check_cache(const Shape &s, const nc_paged4_cache &c) {
    if (!c.k || !c.v || !c.k_scales || !c.v_scales) return NC_ERROR_INVALID_VALUE;
    if (c.k_len < s.cache_len / 2 || c.v_len < s.cache_len / 2 || c.k_scales_len < s.cache_len / 32 || c.v_scales_len < s.cache_len / 32)
        return NC_ERROR_INVALID_VALUE;
    return (address(c.k) | address(c.v)) % 16 ? NC_ERROR_INVALID_VALUE : NC_SUCCESS;
}

struct CacheRanges {
    Range r[4];  // codes of K and V, scales of K and V
};
CacheRanges ranges_of(const Shape &s, const nc_paged4_cache &c) {
    return {{range_of(c.k, s.cache_len / 2, 1), range_of(c.v, s.cache_len / 2, 1), range_of(c.k_scales, s.cache_len / 32, 1),
             range_of(c.v_scales, s.cache_len / 32, 1)}};
}

// Whether a row of K shares memory with one of V, in two pools of units of `unit` values and `bytes` bytes.
bool pools_meet(const Shape &s, const void *k, const void *v, uint64_t unit, uint64_t bytes) {
    const nc_paged_options &o = s.o;
    const uint64_t d = o.head_dim / unit;
    if (!overlap(range_of(k, s.cache_len / unit, bytes), range_of(v, s.cache_len / unit, bytes))) return false;
    Axis cache[] = {{o.num_pages, o.page_stride / unit}, {o.num_kv_heads, o.head_stride / unit}, {o.page_size, o.token_stride / unit}};
    uint64_t unused;
    if (extent(cache, 3, d, &unused)) return true;
    const int64_t apart = (int64_t)(address(v) - address(k));
    return rows_meet(cache, 3, (int64_t)d, apart / (int64_t)bytes);
}

// A cache that is written: its four parts have to be apart.
bool parts_meet(const Shape &s, const nc_paged4_cache &c) {
    const CacheRanges x = ranges_of(s, c);
    for (int i = 0; i < 2; ++i)
        for (int j = 2; j < 4; ++j)
            if (overlap(x.r[i], x.r[j])) return true;
    return pools_meet(s, c.k, c.v, 2, 1) || pools_meet(s, c.k_scales, c.v_scales, 32, 1);
}

// The rows' arguments and grid; *none where there is nothing to do.
int rows_args(const Shape &s, const void *k_rows, uint64_t k_len, const void *v_rows, uint64_t v_len, const int32_t *slots, uint64_t slots_len,
              uint64_t num_rows, const nc_paged4_cache &c, nc_paged4_rows_args *args, uint32_t *grid, uint64_t *rows_len) {
    const nc_paged_options &o = s.o;
    if (num_rows > kMost31) return NC_ERROR_OVERFLOW;
    Axis row[] = {{num_rows, o.row_stride}, {o.num_kv_heads, o.row_head_stride}};
    int st = extent(row, 2, o.head_dim, rows_len);
    if (st) return st;
    if (!k_rows || !v_rows || !slots || k_len < *rows_len || v_len < *rows_len || slots_len < num_rows) return NC_ERROR_INVALID_VALUE;
    if ((address(k_rows) | address(v_rows)) % 2 || address(slots) % 4) return NC_ERROR_INVALID_VALUE;
    nc_paged4_rows_args &a = *args;
    std::memset(&a, 0, sizeof a);
    a.slots = slots;
    a.k = c.k;
    a.v = c.v;
    a.k_scales = c.k_scales;
    a.v_scales = c.v_scales;
    a.row_stride = o.row_stride;
    a.row_head_stride = o.row_head_stride;
    a.page_stride = o.page_stride;
    a.head_stride = o.head_stride;
    a.token_stride = o.token_stride;
    a.num_rows = num_rows;
    a.num_slots = (uint32_t)(o.num_pages * o.page_size);
    a.bf = o.element_type == NC_ELEMENT_BF16;
    a.ps = nc_paged_make_div((uint32_t)o.page_size);
    const uint64_t chunks = o.num_kv_heads * (o.head_dim / 8);
    if (chunks > kMost31 / 2) return NC_ERROR_OVERFLOW;
    a.chunks = nc_paged_make_div((uint32_t)chunks);
    a.chunk_shift = o.head_dim == 32 ? 2 : o.head_dim == 64 ? 3 : 4;
    // a chunk a thread, and no more than 2^23 workgroups
    a.wg_rows = (uint32_t)std::max<uint64_t>(std::max<uint64_t>(1, 256 / chunks), (num_rows + (1u << 23) - 1) >> 23);
    if (a.wg_rows * chunks > kMost31) return NC_ERROR_OVERFLOW;
    *grid = (uint32_t)((num_rows + a.wg_rows - 1) / a.wg_rows);
    return NC_SUCCESS;
}

// The mass of a call, and how long it has to be.
int check_mass(const Shape &s, const nc_paged_mass &m, uint64_t *stride, uint64_t *len) {
    const uint64_t tokens = s.o.max_pages * s.o.page_size;
    *stride = m.mass_stride ? m.mass_stride : tokens;
    if (*stride > kMostElements) return NC_ERROR_OVERFLOW;
    Axis row[] = {{s.o.num_seqs, *stride}};
    int st = extent(row, 1, tokens, len);
    if (st) return st;
    return !m.mass || m.mass_len < *len || address(m.mass) % 4 ? NC_ERROR_INVALID_VALUE : NC_SUCCESS;
}

// The second launch of an attention that kept its scores.
int launch_weights(nc_module module, const Shape &s, const DecodePlan &plan, const DecodeTensors &t, float *mass, uint64_t stride, nc_stream stream) {
    nc_paged_mass_args a;
    std::memset(&a, 0, sizeof a);
    a.scores = reinterpret_cast<const float *>(static_cast<char *>(t.workspace) + plan.scores);
    a.row_ml = reinterpret_cast<const float *>(static_cast<char *>(t.workspace) + plan.row_ml);
    a.seq_lens = t.seq_lens;
    a.mass = mass;
    a.score_pitch = plan.score_pitch;
    a.mass_stride = stride;
    a.num_seqs = (uint32_t)s.o.num_seqs;
    a.num_q_heads = (uint32_t)s.o.num_q_heads;
    a.max_tokens = (uint32_t)(s.o.max_pages * s.o.page_size);
    // 256 tokens a workgroup, of as many as the table's row has room for; no more than a few thousand, which then take turns
    const uint64_t chunks = (a.max_tokens + 255ull) / 256, y = std::min<uint64_t>(s.o.num_seqs, 65535);
    const uint64_t x = std::min<uint64_t>(chunks, std::max<uint64_t>(1, 4096 / y));
    return launch(module, kWeights, (uint32_t)x, (uint32_t)y, 256, &a, stream);
}

void more_args(const DecodePlan &plan, const DecodeTensors &t, nc_paged_more_args *m) {
    m->scores = reinterpret_cast<float *>(static_cast<char *>(t.workspace) + plan.scores);
    m->row_ml = reinterpret_cast<float *>(static_cast<char *>(t.workspace) + plan.row_ml);
    m->score_pitch = plan.score_pitch;
}

// Offsets of the eviction's workspace.
struct EvictSpace {
    uint64_t news, olds, first, cuts, taken, read, states, lows, counts, source, kept_mass, bytes;
    uint64_t parts, part;  // 0: one workgroup a request
};
// A table of so many tokens is selected from by parts, unless the requests are so many that this is too many workgroups, most of them for
// requests that are not cut.
constexpr uint64_t kLongTable = 12288, kMostPartWgs = 1u << 16;

EvictSpace evict_space(const Shape &s) {
    const uint64_t seqs = 4 * ((s.o.num_seqs + 3) / 4 * 4), tokens = 4 * s.o.num_seqs * s.o.max_pages * s.o.page_size;
    EvictSpace e;
    e.news = 16;
    e.olds = e.news + seqs;
    e.first = e.olds + seqs;
    e.cuts = e.first + seqs;
    // chains and chunks there may be, in 16 bits, which has more of them
    const uint64_t chains = 2 * s.o.num_kv_heads, chunks = s.o.max_pages * s.o.page_size * (s.o.head_dim / 8) / (NC_PAGED4_MOVE_ROWS * NC_PAGED4_MOVE_THREADS) + 1;
    e.taken = e.cuts + seqs;
    e.read = e.taken + (4 * s.o.num_seqs * chains + 15) / 16 * 16;
    e.states = e.read + (4 * s.o.num_seqs * chains * chunks + 15) / 16 * 16;
    const uint64_t width = s.o.max_pages * s.o.page_size;
    e.part = std::max<uint64_t>(2048, (width + 2048 * NC_PAGED4_MOST_PARTS - 1) / (2048 * NC_PAGED4_MOST_PARTS) * 2048);
    e.parts = (width + e.part - 1) / e.part;
    if (width < kLongTable || s.o.num_seqs * (e.parts + 1) > kMostPartWgs) e.parts = 0;
    e.lows = e.states + (e.parts ? 32 * s.o.num_seqs : 0);
    e.counts = e.lows + (8 * s.o.num_seqs * e.parts + 15) / 16 * 16;
    e.source = e.counts + 4 * s.o.num_seqs * e.parts * NC_PAGED4_BINS;
    // the second pass's counts have the place of what is listed later
    e.kept_mass = e.source + (tokens + 15) / 16 * 16;
    e.bytes = e.kept_mass + std::max(tokens, 4 * s.o.num_seqs * e.parts * NC_PAGED4_BINS);
    return e;
}

constexpr uint64_t kMostEvicted = 1ull << 20;  // requests

// What both evictions have in common. `parts`: the cache's, each of them written.
int evict(nc_module module, const nc_paged_evict_lists &t, const nc_paged_evict_rules *rules, const Shape &s, const Range *parts, int num_parts,
          nc_paged_evict_args *args, nc_stream stream) {
    const nc_paged_options &o = s.o;
    if (!rules || !module || !t.block_table || !t.seq_lens || (!t.free_pages && t.free_len) || !t.cursor || !t.kept_lens || !t.counts || !t.workspace)
        return NC_ERROR_INVALID_VALUE;
    if (o.num_seqs > kMostEvicted || t.free_len > kMost31) return NC_ERROR_OVERFLOW;
    if (!rules->budget || rules->limit < rules->budget || rules->sinks > rules->budget || rules->recent > rules->budget - rules->sinks)
        return NC_ERROR_INVALID_VALUE;
    const EvictSpace space = evict_space(s);
    if (t.table_len < s.table_len || t.lens_len < o.num_seqs || t.kept_len < o.num_seqs || t.cursor_len < 1 || t.counts_len < 4 ||
        t.workspace_bytes < space.bytes)
        return NC_ERROR_INVALID_VALUE;
    if ((address(t.block_table) | address(t.seq_lens) | address(t.free_pages) | address(t.cursor) | address(t.kept_lens) | address(t.counts)) % 4 ||
        address(t.workspace) % 16)
        return NC_ERROR_INVALID_VALUE;
    uint64_t mass_stride = 0, mass_len = 0;
    int st = check_mass(s, t.mass, &mass_stride, &mass_len);
    if (st) return st;
    // Outputs first; a pair may be one and the same buffer only where the header says so.
    const Range rg[] = {range_of(t.kept_lens, o.num_seqs, 4), range_of(t.counts, 4, 4),          range_of(t.mass.mass, mass_len, 4),
                        range_of(t.free_pages, t.free_len, 4), range_of(t.workspace, space.bytes, 1), range_of(t.seq_lens, o.num_seqs, 4),
                        range_of(t.cursor, 1, 4),              range_of(t.block_table, s.table_len, 4)};
    bool bad = false;
    for (int i = 0; i < 5; ++i)
        for (int j = i + 1; j < 8; ++j) {
            if ((i == 0 && j == 5 && t.kept_lens == t.seq_lens) || (i == 1 && j == 6 && t.counts == t.cursor)) continue;
            bad = bad || overlap(rg[i], rg[j]);
        }
    for (int i = 0; i < num_parts; ++i)
        for (const Range &x : rg) bad = bad || overlap(parts[i], x);
    if (bad) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_evict: an output overlaps another buffer");

    nc_paged_evict_args &a = *args;
    char *work = static_cast<char *>(t.workspace);
    a.table = t.block_table;
    a.seq_lens = t.seq_lens;
    a.cursor = t.cursor;
    a.mass = t.mass.mass;
    a.free_pages = t.free_pages;
    a.kept_lens = t.kept_lens;
    a.counts = t.counts;
    a.totals = reinterpret_cast<int32_t *>(work);
    a.news = reinterpret_cast<int32_t *>(work + space.news);
    a.olds = reinterpret_cast<int32_t *>(work + space.olds);
    a.first = reinterpret_cast<int32_t *>(work + space.first);
    a.cuts = reinterpret_cast<int32_t *>(work + space.cuts);
    a.taken = reinterpret_cast<uint32_t *>(work + space.taken);
    a.read = reinterpret_cast<uint32_t *>(work + space.read);
    a.states = reinterpret_cast<uint32_t *>(work + space.states);
    a.lows = reinterpret_cast<uint32_t *>(work + space.lows);
    a.counts1 = reinterpret_cast<uint32_t *>(work + space.counts);
    a.counts2 = reinterpret_cast<uint32_t *>(work + space.kept_mass);
    a.parts = (uint32_t)space.parts;
    a.part = (uint32_t)space.part;
    a.source = reinterpret_cast<int32_t *>(work + space.source);
    a.kept_mass = reinterpret_cast<float *>(work + space.kept_mass);
    a.table_stride = o.table_stride;
    a.mass_stride = mass_stride;
    a.page_stride = o.page_stride;
    a.head_stride = o.head_stride;
    a.token_stride = o.token_stride;
    a.num_seqs = (uint32_t)o.num_seqs;
    a.num_pages = (uint32_t)o.num_pages;
    a.max_tokens = (uint32_t)(o.max_pages * o.page_size);
    a.free_len = (uint32_t)t.free_len;
    // lengths are below 2^31: a larger limit cuts none, and what belongs to it is then never used
    a.limit = (uint32_t)std::min<uint64_t>(rules->limit, kMost31);
    a.budget = (uint32_t)std::min<uint64_t>(rules->budget, kMost31);
    a.sinks = (uint32_t)std::min<uint64_t>(rules->sinks, kMost31);
    a.recent = (uint32_t)std::min<uint64_t>(rules->recent, kMost31);
    a.ps = nc_paged_make_div((uint32_t)o.page_size);
    a.unit_log2 = (uint32_t)__builtin_ctz((uint32_t)o.head_dim / (a.four ? 32 : 8));
    // Heads that are next to each other share a chain up to 128 bytes.
    a.row_log2 = a.unit_log2;
    if (o.head_stride == o.head_dim)
        while (a.row_log2 < 3 && o.num_kv_heads % (2ull << (a.row_log2 - a.unit_log2)) == 0) ++a.row_log2;
    const uint64_t chains = 2 * (o.num_kv_heads >> (a.row_log2 - a.unit_log2)), size = nc_paged4_chunk(a.row_log2);
    const uint64_t most = std::min<uint64_t>(a.budget, a.max_tokens) - std::min<uint64_t>(a.sinks, a.max_tokens);  // rows of a chain
    const uint64_t chunks = (most + size - 1) / size;
    if (chains * std::max<uint64_t>(chunks, 1) > kMost31 || o.num_seqs * chains > kMost31) return NC_ERROR_OVERFLOW;
    a.chains = (uint32_t)chains;
    a.chunks = (uint32_t)chunks;
    // A workgroup a chunk, but no more than a few thousand, which then take turns: most requests of a batch may not be cut.
    constexpr uint64_t kMoveWgs = 4096;
    a.side_chunks = (uint32_t)std::min(std::max<uint64_t>(chunks, 1), std::max<uint64_t>(1, kMoveWgs / chains));
    a.side_chains = (uint32_t)std::min(o.num_seqs * chains, std::max<uint64_t>(1, kMoveWgs / a.side_chunks));
    a.mass_parts = (a.max_tokens + NC_PAGED4_MASS_PART - 1) / NC_PAGED4_MASS_PART;
    a.mass_wgs = (uint32_t)std::min<uint64_t>(o.num_seqs * a.mass_parts, 512);
    a.tries = nc_internal_evict_tries;
    // Figures of the three ways are at the kernels. A short table's requests are a few waves' work.
    const bool small = a.max_tokens <= 2048;
    if (a.parts) {
        for (uint32_t pass = 0; pass < 4 && !st; ++pass)
            st = launch(module, kPartFirst + pass, (uint32_t)o.num_seqs * (a.parts + (pass == 0 ? 1 : 0)), 1, 512, &a, stream);
    } else {
        st = launch(module, small ? kSelectShort : kSelect, (uint32_t)o.num_seqs, 1, small ? 512 : 1024, &a, stream);
    }
    if (st) return st;
    return launch(module, kMove, a.mass_wgs + (chunks ? a.side_chunks * a.side_chains : 0), 1, NC_PAGED4_MOVE_THREADS, &a, stream);
}

}  // namespace

extern "C" {

int nc_paged4_validate(const nc_paged_options *opts) {
    Shape s;
    return resolve4(opts, &s);
}

int nc_paged4_append(nc_module module, const nc_paged4_append_buffers *buffers, const nc_paged_options *opts, nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged4_append_buffers &t = *buffers;
    Shape s;
    int st = resolve4(opts, &s);
    if (!st && !module) st = NC_ERROR_INVALID_VALUE;
    if (!st) st = check_cache(s, t.cache);
    if (st) return st;
    if (parts_meet(s, t.cache)) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged4_append: parts of the cache share memory");
    if (t.num_rows == 0) return NC_SUCCESS;
    nc_paged4_rows_args a;
    uint32_t grid = 0;
    uint64_t rows_len = 0;
    st = rows_args(s, t.k_rows, t.k_rows_len, t.v_rows, t.v_rows_len, t.slots, t.slots_len, t.num_rows, t.cache, &a, &grid, &rows_len);
    if (st) return st;
    const Range ins[] = {range_of(t.k_rows, rows_len, 2), range_of(t.v_rows, rows_len, 2), range_of(t.slots, t.num_rows, 4)};
    for (const Range &x : ranges_of(s, t.cache).r)
        for (const Range &y : ins)
            if (overlap(x, y)) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged4_append: the rows overlap the cache");
    a.k_in = t.k_rows;
    a.v_in = t.v_rows;
    return launch(module, kAppend, grid, 1, 256, &a, stream);
}

int nc_paged4_read(nc_module module, const nc_paged4_read_buffers *buffers, const nc_paged_options *opts, nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged4_read_buffers &t = *buffers;
    Shape s;
    int st = resolve4(opts, &s);
    if (!st && !module) st = NC_ERROR_INVALID_VALUE;
    if (!st) st = check_cache(s, t.cache);
    if (st || t.num_rows == 0) return st;
    nc_paged4_rows_args a;
    uint32_t grid = 0;
    uint64_t rows_len = 0;
    st = rows_args(s, t.k_rows, t.k_rows_len, t.v_rows, t.v_rows_len, t.slots, t.slots_len, t.num_rows, t.cache, &a, &grid, &rows_len);
    if (st) return st;
    const Range outs[] = {range_of(t.k_rows, rows_len, 2), range_of(t.v_rows, rows_len, 2)};
    bool bad = false;
    for (const Range &x : outs) {
        for (const Range &y : ranges_of(s, t.cache).r) bad = bad || overlap(x, y);
        bad = bad || overlap(x, range_of(t.slots, t.num_rows, 4));
    }
    if (overlap(outs[0], outs[1])) {  // interleaved, if no row of one is part of a row of the other
        Axis row[] = {{t.num_rows, s.o.row_stride}, {s.o.num_kv_heads, s.o.row_head_stride}};
        uint64_t unused;
        const int64_t apart = (int64_t)(address(t.v_rows) - address(t.k_rows)) / 2;
        bad = bad || extent(row, 2, s.o.head_dim, &unused) || rows_meet(row, 2, (int64_t)s.o.head_dim, apart);
    }
    if (bad) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged4_read: the rows overlap another buffer");
    a.k_out = t.k_rows;
    a.v_out = t.v_rows;
    return launch(module, kRead, grid, 1, 256, &a, stream);
}

uint64_t nc_paged_mass_workspace_bytes(const nc_paged_options *opts) {
    Shape s;
    return resolve(opts, &s) ? 0 : decode_plan(s, true, false, true).bytes;
}

uint64_t nc_paged4_workspace_bytes(const nc_paged_options *opts, int with_mass) {
    Shape s;
    return resolve4(opts, &s) ? 0 : decode_plan(s, true, true, with_mass != 0).bytes;
}

uint64_t nc_paged_evict_workspace_bytes(const nc_paged_options *opts) {
    Shape s;
    return resolve(opts, &s) ? 0 : evict_space(s).bytes;
}

int nc_paged_decode_mass(nc_module module, const nc_paged_decode_buffers *buffers, const nc_paged_mass *mass, const nc_paged_options *opts,
                         nc_stream stream) {
    if (!buffers || !mass) return NC_ERROR_INVALID_VALUE;
    const nc_paged_decode_buffers &t = *buffers;
    Shape s;
    int st = resolve(opts, &s);
    if (st) return st;
    const DecodeTensors x = {t.q, t.q_len, t.block_table, t.table_len, t.seq_lens, t.lens_len, t.o, t.o_len, t.workspace, t.workspace_bytes};
    const DecodePlan plan = decode_plan(s, o_is_vec(s, t.o), false, true);
    if (!module || !t.k_cache || !t.v_cache || t.k_len < s.cache_len || t.v_len < s.cache_len) return NC_ERROR_INVALID_VALUE;
    if ((address(t.k_cache) | address(t.v_cache)) % 16) return NC_ERROR_INVALID_VALUE;
    uint64_t stride = 0, len = 0;
    st = check_decode(s, plan, x);
    if (!st) st = check_mass(s, *mass, &stride, &len);
    if (st) return st;
    const Range more[] = {range_of(t.k_cache, s.cache_len, 2), range_of(t.v_cache, s.cache_len, 2), range_of(mass->mass, len, 4)};
    bool bad = decode_overlaps(s, plan, x, more, 3);
    const Range ins[] = {more[0], more[1], range_of(t.q, s.q_len, 2), range_of(t.block_table, s.table_len, 4), range_of(t.seq_lens, s.o.num_seqs, 4)};
    for (const Range &y : ins) bad = bad || overlap(more[2], y);
    if (bad) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_decode_mass: O, the mass or the workspace overlaps another buffer");

    nc_paged_more_args a;
    std::memset(&a, 0, sizeof a);
    decode_args(s, plan, x, t.k_cache, t.v_cache, &a.a);
    more_args(plan, x, &a);
    const uint32_t kernel = kMass + 4 * plan.size + 2 * plan.odd + (s.o.element_type == NC_ELEMENT_BF16 ? 1 : 0);
    st = launch(module, kernel, plan.grid, 1, 64 * NC_PAGED_WAVES, &a, stream);
    return st ? st : launch_weights(module, s, plan, x, mass->mass, stride, stream);
}

int nc_paged4_decode(nc_module module, const nc_paged4_decode_buffers *buffers, const nc_paged_mass *mass, const nc_paged_options *opts,
                     nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged4_decode_buffers &t = *buffers;
    Shape s;
    int st = resolve4(opts, &s);
    if (!st && !module) st = NC_ERROR_INVALID_VALUE;
    if (!st) st = check_cache(s, t.cache);
    if (st) return st;
    const DecodeTensors x = {t.q, t.q_len, t.block_table, t.table_len, t.seq_lens, t.lens_len, t.o, t.o_len, t.workspace, t.workspace_bytes};
    const DecodePlan plan = decode_plan(s, o_is_vec(s, t.o), true, mass != nullptr);
    uint64_t stride = 0, len = 0;
    st = check_decode(s, plan, x);
    if (!st && mass) st = check_mass(s, *mass, &stride, &len);
    if (st) return st;
    const CacheRanges cache = ranges_of(s, t.cache);
    const Range m = range_of(mass ? mass->mass : nullptr, len, 4);
    const Range more[] = {cache.r[0], cache.r[1], cache.r[2], cache.r[3], m};
    bool bad = decode_overlaps(s, plan, x, more, 5);
    const Range ins[] = {cache.r[0], cache.r[1], cache.r[2], cache.r[3], range_of(t.q, s.q_len, 2), range_of(t.block_table, s.table_len, 4),
                         range_of(t.seq_lens, s.o.num_seqs, 4)};
    for (const Range &y : ins) bad = bad || overlap(m, y);
    if (bad) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged4_decode: O, the mass or the workspace overlaps another buffer");

    nc_paged_more_args a;
    std::memset(&a, 0, sizeof a);
    decode_args(s, plan, x, t.cache.k, t.cache.v, &a.a);
    a.k_scales = t.cache.k_scales;
    a.v_scales = t.cache.v_scales;
    a.bf = s.o.element_type == NC_ELEMENT_BF16;
    if (mass) more_args(plan, x, &a);
    a.values = s.cache_len;
    a.next_least = plan.next_least;
    // Column groups: 4, 2 or one. 64 requests of 8000 over 8 heads of 64 with 4 query heads each take 65.7, 70.6 and 75.6 us, with 8 each 69.3
    // and 76.0 (two groups, one); 16 of 1000 over 8 of 128 14.3, 14.5 and 14.4.
    const uint32_t pack = s.group <= 4 ? 2 : s.group <= 8 ? 1 : 0;
    st = launch(module, kDecode4 + 12 * (plan.size - 1) + 4 * pack + (mass ? 2 : 0) + plan.odd, plan.grid, 1, 64 * NC_PAGED_WAVES, &a, stream);
    return st || !mass ? st : launch_weights(module, s, plan, x, mass->mass, stride, stream);
}

int nc_paged_evict(nc_module module, const nc_paged_evict_buffers *buffers, const nc_paged_evict_rules *rules, const nc_paged_options *opts,
                   nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged_evict_buffers &t = *buffers;
    Shape s;
    int st = resolve(opts, &s);
    if (st) return st;
    if (!t.k_cache || !t.v_cache || t.k_len < s.cache_len || t.v_len < s.cache_len) return NC_ERROR_INVALID_VALUE;
    if ((address(t.k_cache) | address(t.v_cache)) % 16) return NC_ERROR_INVALID_VALUE;
    if (pools_meet(s, t.k_cache, t.v_cache, 1, 2)) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged_evict: rows of K and V share memory");
    const Range parts[] = {range_of(t.k_cache, s.cache_len, 2), range_of(t.v_cache, s.cache_len, 2)};
    nc_paged_evict_args a;
    std::memset(&a, 0, sizeof a);
    a.k = reinterpret_cast<uint8_t *>(t.k_cache);
    a.v = reinterpret_cast<uint8_t *>(t.v_cache);
    return evict(module, t.lists, rules, s, parts, 2, &a, stream);
}

int nc_paged4_evict(nc_module module, const nc_paged4_evict_buffers *buffers, const nc_paged_evict_rules *rules, const nc_paged_options *opts,
                    nc_stream stream) {
    if (!buffers) return NC_ERROR_INVALID_VALUE;
    const nc_paged4_evict_buffers &t = *buffers;
    Shape s;
    int st = resolve4(opts, &s);
    if (!st) st = check_cache(s, t.cache);
    if (st) return st;
    if (parts_meet(s, t.cache)) return nc_internal_fail(NC_ERROR_INVALID_VALUE, "nc_paged4_evict: parts of the cache share memory");
    nc_paged_evict_args a;
    std::memset(&a, 0, sizeof a);
    a.k = t.cache.k;
    a.v = t.cache.v;
    a.k_scales = t.cache.k_scales;
    a.v_scales = t.cache.v_scales;
    a.four = 1;
    return evict(module, t.lists, rules, s, ranges_of(s, t.cache).r, 4, &a, stream);
}

}  // extern "C"
