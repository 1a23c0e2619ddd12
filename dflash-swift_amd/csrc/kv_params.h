/*
 * kv_params.h -- kernel arguments shared by the cache, attention and log-probability kernels
 * and the host code that launches them.
 */
#ifndef DFQ_KV_PARAMS_H
#define DFQ_KV_PARAMS_H

#include <stdint.h>

#define DFQ_KV_THREADS 256

/* One quantised array pair of a cache (K or V), [slots][heads][capacity][..]. */
struct KvArrays {
    uint32_t* codes;
    uint16_t* scales;
    uint16_t* biases;
};

/* Division of 0 .. 2^31 - 1 by a number that the host knows: with l the number's bits rounded up
 * and mul = floor(2^32 (2^l - by) / by) + 1, n / by = (n + floor(n mul / 2^32)) >> l. */
struct Divisor {
    uint32_t by, mul;
    int shift;
};

struct KvAppendParams {
    KvArrays out[2];         /* K, V                                             */
    const uint16_t* in[2];   /* rows [batch * rows], row_stride elements apart   */
    const int32_t* starts;   /* first position of each sequence, added to start  */
    int64_t row_stride;
    int start, rows, heads, capacity;
};

struct KvReadParams {
    KvArrays in[2];
    void* out[2];            /* dense [batch][rows][heads][dim], NULL: not wanted */
    const int32_t* starts;
    int start, rows, heads, capacity;
};

struct KvAttnParams {
    KvArrays prefix[2];      /* K, V of the shared prefix (slot 0)               */
    KvArrays own[2];         /* K, V of the sequences' own caches                */
    const uint16_t* q;
    uint16_t* y;
    float* lse;              /* [batch][rows][q_heads] or NULL                   */
    const int32_t* lengths;  /* own tokens of each sequence, the block's included */
    const uint32_t* tree;    /* [batch][rows] row masks or NULL (a chain)        */
    /* The parts of a row from each range of tokens: [slot][head][row] pairs (offset, sum) and
     * [slot][head][row][dim] sums in the kernel's channel order; slots are the prefix's ranges,
     * then the own caches' ranges. */
    float* part_ml;
    float* part_o;
    int64_t q_stride;
    int prefix_length, prefix_capacity, own_capacity, max_length;
    int batch;
    Divisor rows, heads, group;             /* group: query heads of a K/V head         */
    Divisor prefix_splits, prefix_blocks;   /* ranges of the prefix; blocks of its rows */
    Divisor own_splits, own_blocks;         /* the same for one sequence                */
    Divisor own_jobs;                       /* the product of those two                 */
    int join_rows;           /* rows that a workgroup joins: 1 or (a wave a row) 4 */
    float scale_log2e;       /* softmax scale * log2(e)                          */
};

struct LogprobParams {
    const void* logits;
    const int32_t* tokens;   /* or NULL */
    float* logprobs;
    float* entropy;
    int32_t* top_tokens;
    float* top_logprobs;
    uint64_t* part_keys;     /* [row][part][top]: its best order keys, 0 where it has fewer */
    float* part_sums;        /* [row][part][4]: maximum, sum, entropy sum                   */
    int64_t row_stride;
    int rows, vocab, top;
    int splits;              /* workgroups, and parts, a row                                */
};

#endif
