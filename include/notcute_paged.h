/*
 * notcute_paged.h — C ABI of the paged key-value cache: what follows the flash forward of
 * notcute_flash.h once a prompt is in, on MI355X (gfx950).
 *
 *   nc_paged_build    block tables, slot map and row offsets from the requests' lengths
 *   nc_paged_append   new K and V rows into the cache's pages
 *   nc_paged_decode   attention of one new token per request over its pages
 *
 * An extension: the reference has no cache. Conventions as in notcute_flash.h: nc_status return codes,
 * plain device pointers with element counts, f16 (or bf16) bit patterns as uint16_t, O in f32,
 * asynchronous on the given stream. A call's tensors come as one block of pointers and lengths in elements,
 * which it reads before it returns. No call allocates, synchronises or copies; every one may be captured
 * into a HIP graph (nc_paged_build may be two launches, the others are one). `module` is one from
 * nc_module_load_embedded; the first of these calls through it loads the kernels (about 1.4 ms, once).
 *
 * The cache. K and V are each a pool of `num_pages` pages of `page_size` tokens. The row of token t and
 * key head h in page p starts at element p*page_stride + h*head_stride + t*token_stride and holds
 * head_dim elements. By default a page holds its heads one after the other, [page][head][token][dim];
 * [page][token][head][dim] is token_stride = num_kv_heads*head_dim, head_stride = head_dim;
 * K and V may also be interleaved in one allocation. A token's slot
 * is page*page_size + place in the page.
 *
 * The block table. Row r of it lists the pages of request r: token j of the request is at place
 * j % page_size of page table[r][j / page_size]. Entries past the request's length are never read.
 * Pages may be shared between requests that only read them.
 *
 * What device memory holds is not checked on the host, so the kernels check it: an entry outside
 * [0, num_pages) stands for absent keys, a length is cut to what the table's row can hold (negative: 0),
 * a slot outside the pool is skipped.
 */
#ifndef NOTCUTE_PAGED_H
#define NOTCUTE_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "notcute_flash.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct nc_paged_options {
    uint64_t num_seqs;     /* requests: rows of the block table */
    uint64_t num_q_heads;  /* a multiple of num_kv_heads: query head i reads key head i / (num_q_heads/num_kv_heads) */
    uint64_t num_kv_heads;
    uint64_t head_dim;     /* 16, 32, 64 or 128 */
    uint64_t page_size;    /* tokens of a page, any number from 1 */
    uint64_t num_pages;    /* pages of the pool */
    uint64_t max_pages;    /* width of the block table */
    /* Strides in elements; 0 takes the packed value. */
    uint64_t table_stride;    /* 0 => max_pages */
    uint64_t page_stride;     /* 0 => the larger of num_kv_heads*head_stride and page_size*token_stride */
    uint64_t head_stride;     /* 0 => page_size * token_stride */
    uint64_t token_stride;    /* 0 => head_dim */
    uint64_t row_stride;      /* nc_paged_append's K and V rows: 0 => num_kv_heads * row_head_stride */
    uint64_t row_head_stride; /* 0 => head_dim */
    uint64_t q_stride;        /* Q of one request: 0 => num_q_heads * q_head_stride */
    uint64_t q_head_stride;   /* 0 => head_dim */
    uint64_t o_stride;        /* O of one request: 0 => num_q_heads * o_head_stride */
    uint64_t o_head_stride;   /* 0 => head_dim */
    float scale;              /* of the scores; nc_paged_options_init leaves 0 */
    uint32_t element_type;    /* NC_ELEMENT_F16 or NC_ELEMENT_BF16: Q, the new rows and the cache */
} nc_paged_options;

/* All fields zero but num_seqs = num_q_heads = num_kv_heads = max_pages = 1. */
void nc_paged_options_init(nc_paged_options *opts);

/* NC_ERROR_INVALID_VALUE: a count that is 0, query heads that are no multiple of the key heads, another
 * head_dim or element_type, a stride that makes two rows overlap, a cache stride that is no multiple of
 * 8 elements (16 bytes). NC_ERROR_OVERFLOW: more than 2^31 - 1 slots in the pool, tokens in a table row,
 * requests or outputs of a request (num_q_heads * head_dim); more than 2^30 blocks of keys to share out
 * (for each request, key head and part of up to 64 of the key head's query heads, a block for every 32 tokens
 * of the table's row and two more are always within what counts); a tensor past 2^60 elements. */
int nc_paged_validate(const nc_paged_options *opts);

/* Block tables, slot map and row offsets of one step, from the requests' lengths.
 *
 * Request r has cached_lens[r] = c tokens in the cache, in ceil(c/page_size) pages that its table row
 * lists, and new_lens[r] = n tokens to come (negative lengths count as 0). The step's new rows stand one
 * request after the other: row_offsets[r] is the first row of request r, row_offsets[num_seqs] their number.
 * The pages that the new tokens need beyond those held are taken from free_pages, from cursor[0] on, in
 * the requests' order, and entered into the table row; slots[row] is each new row's slot, and -1 in the
 * places behind the last row. seq_lens[r] = c + n.
 *
 * A request that does not fit is refused as a whole: its slots are -1, seq_lens[r] = c, it takes no page and
 * its table row stays as it is. That is one that needs more pages than the table's width or than are left
 * on the list behind what the requests before it asked for, or whose rows go past the slot map
 * (row_offsets are cut to its length). A listed page outside [0, num_pages) gives slots of -1.
 *
 * counts[0] = cursor + pages taken, counts[1] = rows, counts[2] = pages taken, counts[3] = requests refused.
 *
 * seq_lens may be cached_lens itself and counts may be cursor itself (advanced in place, so that one
 * captured step can be replayed); no other output may overlap another buffer (NC_ERROR_INVALID_VALUE).
 * Lengths in elements: cached_len, new_len, seq_len >= num_seqs; offsets_len >= num_seqs + 1; table_len >=
 * (num_seqs - 1)*table_stride + max_pages; counts_len >= 4, cursor_len >= 1; slots_len places are written
 * (0 to 2^31 - 1 of them, slots may be NULL for 0), free_len may be 0. */
typedef struct nc_paged_build_buffers {
    const int32_t *cached_lens;
    uint64_t cached_len;
    const int32_t *new_lens;
    uint64_t new_len;
    const int32_t *free_pages;
    uint64_t free_len;
    const int32_t *cursor;
    uint64_t cursor_len;
    int32_t *block_table;
    uint64_t table_len;
    int32_t *seq_lens;
    uint64_t seq_len;
    int32_t *row_offsets;
    uint64_t offsets_len;
    int32_t *slots;
    uint64_t slots_len;
    int32_t *counts;
    uint64_t counts_len;
} nc_paged_build_buffers;
int nc_paged_build(nc_module module, const nc_paged_build_buffers *buffers, const nc_paged_options *opts,
                   nc_stream stream);

/* K and V rows into the cache: row i (element i*row_stride + h*row_head_stride of k_rows and v_rows, at any
 * element alignment) goes to slot slots[i], for the num_rows first rows; a slot outside the pool (-1) is
 * skipped. Slots of one call are distinct: of two rows with the same slot, either may be kept, element by
 * element. The caches are 16-byte aligned, do not overlap the rows, and no row of the one shares an element
 * with a row of the other (NC_ERROR_INVALID_VALUE). num_rows = 0 does nothing. */
typedef struct nc_paged_append_buffers {
    const uint16_t *k_rows;
    uint64_t k_rows_len;
    const uint16_t *v_rows;
    uint64_t v_rows_len;
    const int32_t *slots;
    uint64_t slots_len;
    uint16_t *k_cache;
    uint64_t k_len;
    uint16_t *v_cache;
    uint64_t v_len;
    uint64_t num_rows;
} nc_paged_append_buffers;
int nc_paged_append(nc_module module, const nc_paged_append_buffers *buffers, const nc_paged_options *opts,
                    nc_stream stream);

/* Device memory that nc_paged_decode needs for these options (0 when they are invalid). The caller zeroes
 * it once before its first use; every launch that runs to its end leaves it ready for the next, of any
 * options that need no more. Launches that overlap in time need workspaces of their own (two streams, or two
 * graphs that may run at once). */
uint64_t nc_paged_workspace_bytes(const nc_paged_options *opts);

/* O[r][i] = sum_j p_j V[j] over the seq_lens[r] tokens j of request r, p = softmax_j(scale * Q[r][i] . K[j]),
 * for every query head i. Scores, maxima, exponentials and sums are f32. The weights enter the product with V as the sum of
 * two (f16) or three (bf16) 16-bit numbers, which is the f32 weight to 2^-21 or better for weights down to 2^-29 (f16) or
 * 2^-70 (bf16) of the largest one, and below that off by at most 2^-51 or 2^-93 of the largest one. In bf16, what is
 * below 2^-94, of V or of a weight (over the largest one) times V, may count as 0. A request of length 0, one whose pages
 * are all absent and one whose scores are all -infinity get zeros. A NaN among the keys that count gives NaN, and so does a
 * score of +infinity. An infinite V among them gives that infinity, and NaN together with the other one or where its weight
 * is below 2^-39 (f16) or 2^-93 (bf16) of the largest one. What lies elsewhere in the pools may be anything. Q at any element
 * alignment, O at any float; caches and workspace 16-byte aligned. O and the workspace overlap nothing else
 * (NC_ERROR_INVALID_VALUE). Rows of O behind the last request are not touched. How the keys are split over
 * workgroups follows the lengths of all requests, so a request's rounding may differ with its neighbours;
 * equal calls give equal bits. */
typedef struct nc_paged_decode_buffers {
    const uint16_t *q;
    uint64_t q_len;
    const uint16_t *k_cache;
    uint64_t k_len;
    const uint16_t *v_cache;
    uint64_t v_len;
    const int32_t *block_table;
    uint64_t table_len;
    const int32_t *seq_lens;
    uint64_t lens_len;
    float *o;
    uint64_t o_len;
    void *workspace;
    uint64_t workspace_bytes;
} nc_paged_decode_buffers;
int nc_paged_decode(nc_module module, const nc_paged_decode_buffers *buffers, const nc_paged_options *opts,
                    nc_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* NOTCUTE_PAGED_H */
