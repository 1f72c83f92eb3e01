/*
 * notcute_paged4.h — C ABI of a smaller paged key-value cache on MI355X (gfx950): fewer bits a value, fewer tokens a request.
 *
 *   nc_paged4_append       new K and V rows into pages of 4 bits
 *   nc_paged4_read         K and V rows out of them
 *   nc_paged4_decode       attention of one new token per request over its pages of 4 bits
 *   nc_paged_decode_mass   nc_paged_decode, and every cached token's share of the weights added up
 *   nc_paged_evict         requests that are too long keep their first, their last and their heaviest tokens;
 *   nc_paged4_evict        in 16 bits and in 4
 *
 * An extension: the reference has no cache. Conventions and options are those of notcute_paged.h, whose block tables
 * (nc_paged_build) serve both kinds of cache. Every call may be captured into a HIP graph; nc_paged_decode_mass,
 * nc_paged4_decode with a mass and the evictions are two launches, or an eviction five where the table is for 12288 tokens and more and the
 * requests are not thousands (num_seqs * (parts + 1) of at most 65536, parts of 2048 tokens or a 64th); the others are one. The first of these calls through a module loads their kernels (about
 * 2.5 ms, once).
 *
 * A cache in 4 bits. K and V are each a pool of codes, two values a byte (the value of the even place in the low half), and a
 * pool of scales, a byte for every 32 values of a row (the microscaling format MXFP4: e2m1 values, e8m0 scales). A code is a
 * sign (bit 3) and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale byte b stands for 2^(b - 127), and 255 for a group of NaN. (Values
 * of 2^128 and more, of bytes 253 and 254, count as infinite in V: O is infinite or NaN then. The append writes none.) The
 * strides of the options count values: the value at element e of the pool (notcute_paged.h) is in byte e / 2 of the codes and has the
 * scale at e / 32. They are multiples of 32, and head_dim is 32, 64 or 128. element_type is the type of Q and of the rows.
 */
#ifndef NOTCUTE_PAGED4_H
#define NOTCUTE_PAGED4_H

#include "notcute_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A cache in 4 bits: codes 16-byte aligned, scales at any byte; lengths in bytes. K and V may be interleaved as those of a
 * 16-bit cache. */
typedef struct nc_paged4_cache {
    uint8_t *k;
    uint64_t k_len;
    uint8_t *v;
    uint64_t v_len;
    uint8_t *k_scales;
    uint64_t k_scales_len;
    uint8_t *v_scales;
    uint64_t v_scales_len;
} nc_paged4_cache;

/* What nc_paged_validate refuses, another head_dim and a cache stride that is no multiple of 32
 * (NC_ERROR_INVALID_VALUE), a pool of 2^37 values or more (NC_ERROR_OVERFLOW). */
int nc_paged4_validate(const nc_paged_options *opts);

/* K and V rows into the cache, as nc_paged_append: row i to slot slots[i], for the num_rows first rows; a slot outside the pool is
 * skipped, and the slots of one call are distinct. Every 32 values of a row get the scale 2^k, k the least whole number with
 * max |x| <= 7 2^k (so that the largest value is off by at most half a step), but at least -23 and at most 13 for f16 rows, at
 * least -125 and at most 125 for bf16 rows; a value x becomes the code next to x / 2^k, of two as near the even one, and the largest
 * code where it lies above that. A group that holds a NaN or an infinity gets the scale byte 255 and codes of 0. The rows overlap no
 * part of the cache, codes and scales do not overlap, and no row of K shares a byte with one of V (NC_ERROR_INVALID_VALUE).
 * num_rows = 0 does nothing. */
typedef struct nc_paged4_append_buffers {
    const uint16_t *k_rows;
    uint64_t k_rows_len;
    const uint16_t *v_rows;
    uint64_t v_rows_len;
    const int32_t *slots;
    uint64_t slots_len;
    nc_paged4_cache cache;
    uint64_t num_rows;
} nc_paged4_append_buffers;
int nc_paged4_append(nc_module module, const nc_paged4_append_buffers *buffers, const nc_paged_options *opts, nc_stream stream);

/* The rows at slots[0..num_rows-1] as dense rows of element_type (options' row_stride and row_head_stride, at any element
 * alignment). nc_flash_launch takes such rows of a prompt that goes on behind a cached one where head_dim is 32 or 64 and every query head
 * has a key head of its own; it is a square forward, so Q has the cached positions too, and their outputs are computed again. Values are exact where the type holds them,
 * as it does for rows that nc_paged4_append wrote from the same type; the row of a slot outside the pool is zeros. A slot
 * may be listed more than once. The rows overlap neither the cache, nor the slots, nor each other (NC_ERROR_INVALID_VALUE; K's and
 * V's may be interleaved as long as no row of one is part of a row of the other). */
typedef struct nc_paged4_read_buffers {
    nc_paged4_cache cache;
    const int32_t *slots;
    uint64_t slots_len;
    uint16_t *k_rows;
    uint64_t k_rows_len;
    uint16_t *v_rows;
    uint64_t v_rows_len;
    uint64_t num_rows;
} nc_paged4_read_buffers;
int nc_paged4_read(nc_module module, const nc_paged4_read_buffers *buffers, const nc_paged_options *opts, nc_stream stream);

/* Masses: a row of floats per request, one per token of the table's row: mass[r*mass_stride + j] of token j. mass_stride 0 is
 * max_pages*page_size, the least that is accepted where there are several requests. */
typedef struct nc_paged_mass {
    float *mass;
    uint64_t mass_len;
    uint64_t mass_stride;
} nc_paged_mass;

/* nc_paged_decode, and mass[r][j] += sum over all query heads of p_j for every token j of request r (those behind its last token
 * stay as they are; a request that gets zeros for O adds nothing, one with a score that is NaN or +infinity adds NaN). The sum over the
 * heads is f32, in a fixed order. Clear a request's row when it begins, and nc_paged_evict keeps it in step. Only these calls add
 * weights: those of a prompt's own queries are not in it, so that right behind a prompt all masses are 0 and an eviction keeps the earlier
 * tokens. Over 16 bits heads are taken each for itself: where nc_paged_decode takes neighbouring heads, or a wave a short head, this
 * is slower by more than the scores. The workspace is as
 * nc_paged_decode's, but larger by the scores, 4 bytes for every request, query head and token of the table's row
 * (nc_paged_mass_workspace_bytes). The mass overlaps nothing else (NC_ERROR_INVALID_VALUE). */
uint64_t nc_paged_mass_workspace_bytes(const nc_paged_options *opts);
int nc_paged_decode_mass(nc_module module, const nc_paged_decode_buffers *buffers, const nc_paged_mass *mass,
                         const nc_paged_options *opts, nc_stream stream);

/* nc_paged_decode over a cache in 4 bits. Scores are f32 sums of exact products but for Q: every value of it enters as the sum of
 * four 8-bit or five 6-bit numbers, off by at most 2^-25 of the largest of its 32 (dims 0..31, 32..63, ...) or 2^-130, and not at all where it
 * is above 2^-14 of that in f16, 2^-17 in bf16. The weights enter the product with V as three bf16 parts, as nc_paged_decode's for bf16. A
 * query that is not finite gives NaN, and so do keys that count whose scale byte is 255, in K or in V. A `mass` that is not NULL adds the weights up as nc_paged_decode_mass
 * does. Workspace: nc_paged4_workspace_bytes, with_mass 1 for calls with a mass. */
typedef struct nc_paged4_decode_buffers {
    const uint16_t *q;
    uint64_t q_len;
    nc_paged4_cache cache;
    const int32_t *block_table;
    uint64_t table_len;
    const int32_t *seq_lens;
    uint64_t lens_len;
    float *o;
    uint64_t o_len;
    void *workspace;
    uint64_t workspace_bytes;
} nc_paged4_decode_buffers;
uint64_t nc_paged4_workspace_bytes(const nc_paged_options *opts, int with_mass);
int nc_paged4_decode(nc_module module, const nc_paged4_decode_buffers *buffers, const nc_paged_mass *mass,
                     const nc_paged_options *opts, nc_stream stream);

/* Eviction by accumulated weight (whose time grows with the square of the requests that are cut where they are thousands: 4096 of 20 tokens
 * 54 us, 16384 0.28 ms, 65536 2.7 ms). A request of more than `limit` tokens keeps `budget` of them: its first `sinks`, its last
 * `recent`, and of the others those with the largest mass (of equal ones the earlier; a NaN counts as the largest). */
typedef struct nc_paged_evict_rules {
    uint64_t limit;  /* at least budget */
    uint64_t budget; /* at least 1 */
    uint64_t sinks;
    uint64_t recent; /* sinks + recent at most budget */
} nc_paged_evict_rules;

/* The tokens that stay are moved together at the front, in their order, within the request's own pages: K, V and masses (those
 * behind the last one become 0). kept_lens[r] is the new length, the old one (cut to the table's row, negative: 0) where nothing
 * was evicted. The pages behind the new length go back to the list that nc_paged_build takes pages from: free_pages[cursor - n..cursor - 1]
 * are the n pages that became free, in the requests' order and the tables', entries outside the pool among them. Those that find no place on the list (a cursor below n, or
 * beyond free_len) are lost. The tables are not changed: what they list behind the new length is the list's.
 *
 * counts[0] = cursor - n (at least 0), counts[1] = requests cut, counts[2] = n, counts[3] = tokens evicted. counts[1] is -1 where rows were
 * not moved because another call has changed the workspace meanwhile: the cut requests' rows are lost then.
 *
 * kept_lens may be seq_lens itself and counts may be cursor itself; apart from that no output overlaps another buffer
 * (NC_ERROR_INVALID_VALUE). A page of a request that is cut belongs to it alone: rows of pages that two requests share, or that one lists
 * twice, may be moved in any order. A row on a page outside the pool is not moved, nor is one moved there. Lengths in elements as for the
 * other calls; counts_len >= 4, cursor_len >= 1; workspace 16-byte aligned, nc_paged_evict_workspace_bytes, which need not be
 * cleared; calls that overlap in time need workspaces of their own (what two that share one leave is undefined, and not always told). At
 * most 2^20 requests (NC_ERROR_OVERFLOW). */
typedef struct nc_paged_evict_lists {
    const int32_t *block_table;
    uint64_t table_len;
    const int32_t *seq_lens;
    uint64_t lens_len;
    nc_paged_mass mass;
    int32_t *free_pages;
    uint64_t free_len;
    const int32_t *cursor;
    uint64_t cursor_len;
    int32_t *kept_lens;
    uint64_t kept_len;
    int32_t *counts;
    uint64_t counts_len;
    void *workspace;
    uint64_t workspace_bytes;
} nc_paged_evict_lists;
typedef struct nc_paged_evict_buffers {
    nc_paged_evict_lists lists;
    uint16_t *k_cache;
    uint64_t k_len;
    uint16_t *v_cache;
    uint64_t v_len;
} nc_paged_evict_buffers;
typedef struct nc_paged4_evict_buffers {
    nc_paged_evict_lists lists;
    nc_paged4_cache cache;
} nc_paged4_evict_buffers;
uint64_t nc_paged_evict_workspace_bytes(const nc_paged_options *opts);
int nc_paged_evict(nc_module module, const nc_paged_evict_buffers *buffers, const nc_paged_evict_rules *rules,
                   const nc_paged_options *opts, nc_stream stream);
int nc_paged4_evict(nc_module module, const nc_paged4_evict_buffers *buffers, const nc_paged_evict_rules *rules,
                    const nc_paged_options *opts, nc_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* NOTCUTE_PAGED4_H */
