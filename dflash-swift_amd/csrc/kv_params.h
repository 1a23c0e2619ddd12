/*
 * kv_params.h -- kernel arguments shared by the cache, attention, log-probability, rotation and
 * sampled-accept kernels and the host code that launches them.
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

/* What a wave of dfq_sample_accept's first kernel makes of its range of a row. */
struct AcceptPart {
    float top;               /* the largest logit; NaN where there is one (T > 0)         */
    uint32_t sum;            /* T > 0: the fp32 sum of e^((x - top) / T), 0 where top is not
                              * finite; T = 0: the first place of top, 2^31 - 1 where all
                              * are NaN                                                   */
};

#define DFQ_ACCEPT_APART 32  /* counters lie a cache line apart                          */
#define DFQ_ACCEPT_PIECES 4  /* 16-byte pieces that a lane takes of a range              */

struct AcceptParams {
    const void* logits;
    const void* draft_logits;   /* or NULL: drafts are certain                     */
    const int32_t* drafts;      /* [batch][rows - 1]                               */
    const int32_t* lengths;     /* drafts of each sequence, or NULL: rows - 1      */
    const float* uniforms;      /* [batch][rows]                                   */
    const float* temperatures;  /* [batch], or NULL: `temperature`                 */
    const float* draft_temperatures;
    int32_t* tokens;            /* [batch][rows]                                   */
    int32_t* accepted;          /* [batch]                                         */
    float* chances;             /* [batch][rows - 1] or NULL                       */
    AcceptPart* parts;          /* [batch][rows, then draft rows][ranges]          */
    uint64_t* sums;             /* [batch][sums_apart]: of units, one or (p - q) six; doubles' bits */
    uint64_t* totals;           /* [batch][chunks][2]: both rows' sums, with draft logits  */
    int32_t* arrived;           /* [batch][DFQ_ACCEPT_APART]: workgroups whose sums are there */
    int64_t batch_stride, row_stride, draft_batch_stride, draft_row_stride;
    double near;                /* how far the fp32 sums' p / q may be off, of itself */
    float temperature, draft_temperature;
    int rows, vocab;
    int jobs;                   /* ranges of all rows                              */
    int units;                  /* 64 lanes' 16 bytes each, of a row               */
    int sums_apart;             /* units, six times that with draft logits         */
    Divisor all_rows, ranges;   /* rows and draft rows of a sequence; ranges a row */
    Divisor chunks;             /* workgroups of a sequence in the second kernel   */
};

#define DFQ_ROPE_DIM 512     /* widest head */
#define DFQ_NORM_SMALL 0x1p-100f   /* mean square and eps from which on fp32 squares serve */

struct RopeTensor {
    const void* in;
    void* out;
    const void* weight;      /* [dim] or NULL                                    */
    int64_t in_batch, in_row, in_head, out_batch, out_row, out_head;   /* elements */
    int heads;
    Divisor slots;           /* of a token: slot s holds heads s, s + slots, ..  */
};

struct RopeParams {
    RopeTensor t[2];         /* queries, keys                                    */
    const uint64_t* turns;   /* [pairs] 2^-64 turns a position                   */
    const int32_t* starts;   /* first position of each sequence, added to start  */
    const int32_t* positions;   /* [batch][rows], in place of those, or NULL     */
    int tokens, start, dim, pairs;
    int q_groups;            /* workgroups of the queries; the keys' come behind */
    int lanes;               /* that hold a head (rotate_heads)                  */
    int inverse, interleaved, weight_f32;
    float amplitude, eps, offset;
    Divisor rows;
};

#endif
