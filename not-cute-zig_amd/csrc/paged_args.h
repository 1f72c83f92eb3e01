// paged_args.h — what the host side (paged.cpp, paged4.cpp) and the kernels (paged.hip, paged4.hip) share: argument blocks and
// the index arithmetic that both sides (and the CPU tests) have to agree on.
#ifndef NOTCUTE_PAGED_ARGS_H
#define NOTCUTE_PAGED_ARGS_H

#include <stdint.h>

#ifdef __HIPCC__
#define NC_HD __host__ __device__ __forceinline__
#else
#define NC_HD inline
#endif

// n / d for 0 <= n < 2^31 by one 32x32 high multiply: with 2^s >= d and magic = ceil(2^(31+s) / d),
// n * magic / 2^(31+s) exceeds n/d by less than n / 2^31 / d < 1/d, so its floor is the quotient.
struct nc_paged_div {
    uint32_t d, magic, shift;
};
inline nc_paged_div nc_paged_make_div(uint32_t d) {
    nc_paged_div r = {d, 0, 0};
    while ((1ull << r.shift) < d) ++r.shift;
    r.magic = (uint32_t)(((1ull << (31 + r.shift)) + d - 1) / d);
    return r;
}
NC_HD uint32_t nc_paged_quot(uint32_t n, nc_paged_div v) {
    return (uint32_t)(((uint64_t)(2u * n) * v.magic) >> 32) >> v.shift;
}

#define NC_PAGED_KERNELS 53u  // kernels of paged.hip
#define NC_PAGED4_KERNELS 62u // and of paged4.hip

struct nc_paged_build_args {
    const int32_t *cached, *fresh, *free_pages, *cursor;
    int32_t *table, *seq_lens, *offsets, *slots, *counts;
    uint64_t table_stride;
    uint32_t num_seqs, width, num_pages, free_len, places;
    uint32_t chunk_rows, chunk_pages; // slots and list places of one workgroup
    uint32_t parts;                   // NC_PAGED_PART_*
    nc_paged_div ps;
};
#define NC_PAGED_PART_PAGES 1u // table entries and slots
#define NC_PAGED_PART_LENS 2u  // lengths, offsets and counts

struct nc_paged_append_args {
    const uint16_t *k_rows, *v_rows;
    const int32_t *slots;
    uint16_t *k, *v;
    uint64_t row_stride, row_head_stride, page_stride, head_stride, token_stride;
    uint64_t num_rows;
    uint32_t num_slots;    // num_pages * page_size
    uint32_t wg_rows;      // rows of one workgroup
    uint32_t chunk_shift;  // log2(head_dim / 8)
    nc_paged_div ps, chunks; // page_size, and num_kv_heads * head_dim / 8
};

// The attention's work is counted in blocks: the keys of one request and key head that a workgroup's four waves
// take in a step. A wave takes step_keys of them for 16 query heads; where a key head has more than 16, two or
// four waves take the same keys for 16 heads each (wave_shift 1 or 2), and past 64 the workgroup's heads count
// as another head. Neighbouring heads (the _next kernels) are shared out in the same way: 1 << wave_shift of them count
// as one, a wave each. Those kernels have the code of both ways and take neighbouring heads where a request is longer than
// NC_PAGED_NEXT_TOKENS: the lengths decide it, not the table's width. In a table of 4096 tokens' pages, neighbouring heads and
// each for itself: 2 requests of 200 over 8 heads of 32 6.4 and 4.7 us, 4 of 300 over 8 of 16 6.8 and 5.5; 8 of 400 over 8 of
// 128 9.4 and 9.5.
#define NC_PAGED_WAVES 4u
#define NC_PAGED_NEXT_TOKENS 512u
// With 5 to 8 query heads a key head, two neighbouring heads' pieces are as large as 16 query heads': a call over a cache in 4 bits takes
// neighbouring heads only from so many units on. Each head for itself, and pairs; requests of tokens over 8 heads, 64 query heads:
//   32 of up to 4000, 64   12.8  14.9 us (fewer units)    64 of 4000, 64      90.4  59.9     one of 120001, 64   49.4  34.0
//   64 of up to 4000, 64   21.5  17.8                     64 of 4000, 128    99.5  80.9     100 of 600, 64      29.7  22.5
//   32 of up to 4000, 128  19.6  21.6 (fewer)             16 of 4000, 64      29.1  21.7     4 of 30000, 32      41.5  30.1
//   4 of 20000, 64         21.2  26.5 and 8 of 16000, 64, 26.4  32.8 (taken all the same: the shares happen to put the heads of the same
//                          keys on one XCD, which so many tokens to a request and a few more do not)
#define NC_PAGED4_WIDE_UNITS 1800u
#define NC_PAGED4_STEP_KEYS 64u // a wave's step over a cache in 4 bits, of any head_dim
NC_HD uint32_t nc_paged_step_keys(uint32_t head_dim) { return head_dim <= 32 ? 64u : 32u; }
NC_HD uint32_t nc_paged_wave_shift(uint32_t group) { return group <= 16 ? 0u : group <= 32 ? 1u : 2u; }
NC_HD uint32_t nc_paged_head_parts(uint32_t group) { return (group + 63u) / 64u; }

// Shares are counted in units: one per block, and before a head's first block so many for what a head costs however
// short it is. Workgroup i takes units [i * each, (i + 1) * each), where `each` is the least that 2^most_log2
// workgroups can do with, and no less than `least`. With one unit a head and with two:
//   33 requests of up to 2047, 16 heads of 32   11.1  11.8 us
//   118 of up to 2719, 3 heads of 32            10.8  11.8
//   16 of 1000, 8 heads of 128                  17.2  16.5
//   64 of up to 16000, 4 heads of 64            29.6  28.6
NC_HD constexpr uint32_t nc_paged_head_units(uint32_t head_dim) { return head_dim <= 32 ? 1u : 2u; }
// Caches in 4 bits, with one unit a head and with two:
//   2 requests of 20000, 8 heads of 64 with 8 query heads each    15.3  16.9 us
//   118 of up to 2719, 3 heads of 32                              11.4  11.9
//   96 of 4000, 8 heads of 64 with 8 query heads each             64.9  60.3 (but 64 ragged ones 19.0  18.5)
//   16 of 4000, 8 heads of 128                                    23.4  21.4
//   one of 30000, 8 heads of 128                                  19.8  18.0
//   40 of up to 1500, 8 heads of 128                              12.8  14.9 (200 of up to 500: 26.9  28.1)
NC_HD constexpr uint32_t nc_paged4_head_units(uint32_t head_dim) { return head_dim <= 64 ? 1u : 2u; }
// A head of no more blocks than this is not split: the workgroup that has its first unit takes all of it. (Of 1: 118
// requests of up to 2719, 3 heads of 32, 10.8 -> 11.1 us; of 4: 12.0, and 4 of 500 over 8 heads of 128 7.6 -> 9.4.)
#define NC_PAGED_WHOLE_BLOCKS 2u
// Heads of this many units on the average are long ones. (From 14 on: 16 requests of 1000 over 8 heads of 128 16.5 -> 17.2 us,
// 200 ragged ones of up to 8000 137 -> 145; from 5 on: no change.)
#define NC_PAGED_LONG_UNITS 8u
NC_HD uint32_t nc_paged_each(uint32_t units, uint32_t most_log2, uint32_t least) {
    const uint32_t each = (units + (1u << most_log2) - 1u) >> most_log2;
    return each < least ? least : each;
}

// Pieces that one workgroup adds up in a round, by their size: of up to 16 KB reading 16 of them takes about as long as
// another round (4: 63 pieces of 1 KB 8.7 -> 10.6 us), of more only 4. A CU reads pieces at a few ten GB/s, so that many or
// large ones have to go to several: one request of 100000 tokens takes 20.5 us with 8 query heads on one key head of 128, and
// 58 with 64. At most NC_PAGED_MAX_WGS pieces are one after NC_PAGED_ROUNDS rounds, and NC_PAGED_MERGE_ROWS holds the rows of
// all that one adds up.
#define NC_PAGED_MAX_WGS 1024u
#define NC_PAGED_ROUNDS 5u
#define NC_PAGED_MERGE_ROWS 1024u
// Pieces of few numbers leave threads over, which take every so many-th one: up to 64 at once while all are within 32 KB.
// 21 pieces of 512 bytes 9.4 -> 8.1 us, 32 of 1 KB no change; but 63 of 1 KB, which pass that, 8.7 -> 9.6.
#define NC_PAGED_MERGE_PIECES 64u
NC_HD bool nc_paged_one_round(uint32_t pieces, uint32_t numbers) {
    return pieces <= NC_PAGED_MERGE_PIECES && pieces * numbers <= 8192u;
}
NC_HD uint32_t nc_paged_fan(uint32_t rows, uint32_t head_dim) { return rows * head_dim <= 4096u ? 16u : 4u; }

struct nc_paged_decode_args {
    const uint16_t *q, *k, *v;
    const int32_t *table, *seq_lens;
    float *o;
    uint32_t *counters; // NC_PAGED_ROUNDS times two per workgroup, all 0 between launches
    float *part_ml;     // per workgroup two pieces of `rows` (max, sum) pairs
    float *part_o;      // per workgroup two pieces of rows x head_dim sums
    uint64_t table_stride, page_stride, head_stride, token_stride, q_stride, q_head_stride, o_stride, o_head_stride;
    uint32_t num_seqs, num_q_heads, num_kv_heads, group; // group = num_q_heads / num_kv_heads
    uint32_t num_pages, max_tokens;                      // max_tokens = max_pages * page_size
    uint32_t group_inverse;                              // q * group_inverse >> 16 is q / group for q < 64, group <= 16
    uint32_t rows;                                       // query heads of a piece: min(group, 64)
    uint32_t wave_shift, head_parts;
    uint32_t long_log2, short_log2, each_least; // workgroups for long heads and for short ones, units of a share
    nc_paged_div heads;                         // num_kv_heads * head_parts
    uint32_t side;                              // _next kernels: wave_shift of neighbouring heads
    uint32_t many;                              // a wave may take a short head for itself
    uint32_t q_vec, o_vec;                               // Q, O rows are 16-byte aligned
    float scale;
    nc_paged_div ps;
};

// Behind these, for caches in 4 bits (k and v are then bytes of two values, the strides still count values) and for kernels that
// keep their scores.
struct nc_paged_more_args {
    nc_paged_decode_args a;
    const uint8_t *k_scales, *v_scales; // a byte for every 32 values
    float *scores;                      // a row of score_pitch per request and query head
    float *row_ml;                      // and its (max, 1 / sum)
    uint64_t score_pitch;
    uint64_t values;                    // of a 4-bit pool
    uint32_t bf;                        // Q is bf16
    uint32_t next_least;                // units that neighbouring heads are for, 4 bits
};

// The divisor d / 2^side where 2^side divides d: the same multiplier, as 2^(31+shift) / d is.
NC_HD nc_paged_div nc_paged_div_by(nc_paged_div v, uint32_t side) {
    nc_paged_div r = {v.d >> side, v.magic, v.shift - side};
    return r;
}

// A length from device memory, cut to what the table's row can hold.
NC_HD uint32_t nc_paged_cut(int32_t len, uint32_t most) {
    const uint32_t n = len < 0 ? 0u : (uint32_t)len;
    return n < most ? n : most;
}

#endif
