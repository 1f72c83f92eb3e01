// paged4_args.h — what paged4.cpp and paged4.hip share beyond paged_args.h: argument blocks of the smaller cache's kernels.
#ifndef NOTCUTE_PAGED4_ARGS_H
#define NOTCUTE_PAGED4_ARGS_H

#include <stdint.h>

#include "paged_args.h"

// Rows into 4-bit pages, and out of them.
struct nc_paged4_rows_args {
    const uint16_t *k_in, *v_in; // rows to be written
    uint16_t *k_out, *v_out;     // or the places of rows that are read
    const int32_t *slots;
    uint8_t *k, *v, *k_scales, *v_scales;
    uint64_t row_stride, row_head_stride, page_stride, head_stride, token_stride;
    uint64_t num_rows;
    uint32_t num_slots;   // num_pages * page_size
    uint32_t wg_rows;     // rows of one workgroup
    uint32_t chunk_shift; // log2(head_dim / 8)
    uint32_t bf;
    nc_paged_div ps, chunks; // page_size, and num_kv_heads * head_dim / 8
};

// Scale bytes that a cache of f16 rows has, and of bf16 rows: the least whose values are multiples of 2^-24 or normal numbers,
// the largest whose values the type holds.
#define NC_PAGED4_LEAST_F16 104
#define NC_PAGED4_MOST_F16 140
#define NC_PAGED4_LEAST_BF16 2
#define NC_PAGED4_MOST_BF16 252

// The weights by token, out of the scores that the attention kept.
struct nc_paged_mass_args {
    const float *scores, *row_ml;
    const int32_t *seq_lens;
    float *mass;
    uint64_t score_pitch, mass_stride;
    uint32_t num_seqs, num_q_heads, max_tokens;
};

// Eviction. The selection leaves, by request, its new length, the first place that another token's row moves to, the source slot
// of every place of the new length and that token's mass; which requests are cut; and the move's counts and flags at 0.
//
// The move's work is counted in chunks: NC_PAGED4_MOVE_ROWS rows a thread of 1 << row_log2 16-byte units each, of one chain: K or V of
// one request's head (or of a few that are next to each other).
struct nc_paged_evict_args {
    const int32_t *table, *seq_lens, *cursor;
    float *mass;
    int32_t *free_pages, *kept_lens, *counts;
    uint8_t *k, *v, *k_scales, *v_scales;
    int32_t *news, *olds, *first, *totals; // workspace: by request; totals: cursor, requests cut
    int32_t *cuts;                         // the requests that are cut
    uint32_t *taken, *read;                // by chain: chunks taken, and by chunk whether its rows have been read
    uint32_t *states, *lows;               // of a selection by parts: by request and pass, and by part
    uint32_t *counts1, *counts2;           // by part, NC_PAGED4_BINS each
    int32_t *source;                       // num_seqs rows of max_tokens
    float *kept_mass;                      // the same
    uint64_t table_stride, mass_stride, page_stride, head_stride, token_stride;
    uint32_t num_seqs, num_pages, max_tokens, free_len;
    uint32_t limit, budget, sinks, recent;
    uint32_t unit_log2, row_log2;          // log2 of a head's 16-byte units (4 bits: of 32 values, and their scale), and of a chain's
    uint32_t chains, chunks;               // chains of a request, most chunks of one
    uint32_t parts, part;                  // parts of a request at most, and their tokens
    uint32_t mass_wgs, mass_parts;         // workgroups that move masses, their parts of a request
    uint32_t side_chains, side_chunks;     // workgroups that move rows: side_chunks for each of side_chains chains at a time
    uint32_t tries;                        // looks at 64 chunks' flags before a wait gives up
    uint32_t four;
    nc_paged_div ps;
};
#define NC_PAGED4_BINS 2048u
#define NC_PAGED4_MOST_PARTS 64u
#define NC_PAGED4_MOVE_THREADS 256u
#define NC_PAGED4_MOVE_ROWS 8u
#define NC_PAGED4_MASS_PART 2048u // masses that a workgroup moves at a time
// Rows of a chunk.
NC_HD uint32_t nc_paged4_chunk(uint32_t row_log2) { return NC_PAGED4_MOVE_ROWS * (NC_PAGED4_MOVE_THREADS >> row_log2); }

#endif
