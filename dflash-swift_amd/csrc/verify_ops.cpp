/*
 * verify_ops.cpp -- the C ABI of the quantised key/value cache, its attention and the log
 * probabilities: argument checks, work splits and launches of kv_cache.hip, kv_attention.hip and
 * logprobs.hip.
 */
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "dflash_qmm.h"
#include "kv_params.h"
#include "verify_ops.h"

#if !defined(DFQ_KV_HSACO_PATH) || !defined(DFQ_LOGPROBS_HSACO_PATH) || \
    !defined(DFQ_ATTN64_HSACO_PATH) || !defined(DFQ_ATTN128_HSACO_PATH) || \
    !defined(DFQ_ATTN256_HSACO_PATH)
#error "DFQ_*_HSACO_PATH must name the gfx950 code objects to embed"
#endif

DFQ_EMBED(dfq_kv_hsaco, DFQ_KV_HSACO_PATH)
DFQ_EMBED(dfq_logprobs_hsaco, DFQ_LOGPROBS_HSACO_PATH)
DFQ_EMBED(dfq_attn64_hsaco, DFQ_ATTN64_HSACO_PATH)
DFQ_EMBED(dfq_attn128_hsaco, DFQ_ATTN128_HSACO_PATH)
DFQ_EMBED(dfq_attn256_hsaco, DFQ_ATTN256_HSACO_PATH)

using namespace dfq;

namespace {

/* One format of a cache: [head_dim 64/128/256][bits 4/8][group 32/64/128][bf16/f16]; groups wider
 * than the head have no kernels. */
struct CacheKernels {
    hipFunction_t append = nullptr, read = nullptr, join = nullptr;
    hipFunction_t attention[2] = {};  // up to 1 and 2 row tiles (see attention_tiles)
    int resident[2] = {};             // their workgroups that a CU holds at once
};

struct VerifyOps : LoadedOps {
    static constexpr OpsGroup kGroup = kVerifyOps;
    hipModule_t kv = nullptr, logprobs = nullptr, attention[3] = {};
    CacheKernels cache[3][2][3][2];
    hipFunction_t logprobs_part[3] = {}, logprobs_join[3] = {};  // [bf16/f16/f32]
    dfq_status resolve();
    ~VerifyOps() override {
        if (kv) (void)hipModuleUnload(kv);
        if (logprobs) (void)hipModuleUnload(logprobs);
        for (hipModule_t m : attention)
            if (m) (void)hipModuleUnload(m);
    }
};

/* The most tiles of 16 rows that attention kernels take in one pass.  Two read and unpack the
 * codes once for both: 16 sequences of 8 rows of 40 heads over a shared 16384-token prefix take
 * 102 us, one tile 119.  At heads of 256 their outputs leave a CU room for one workgroup of two
 * tiles and two of one: 16 rows of 16 heads over 16000 tokens 32.5 us against 26.1, so there it
 * is one.  Three and four would take 103 and 137 KB of LDS at heads of 128, a workgroup a CU. */
int attention_tiles(int dim) { return dim == 256 ? 1 : 2; }

dfq_status VerifyOps::resolve() {
    VerifyOps* const o = this;
    static const char* kDt[3] = {"bf16", "f16", "f32"};
    hipError_t e;
    if ((e = hipModuleLoadData(&o->kv, dfq_kv_hsaco)) != hipSuccess)
        return hip_error(e, "hipModuleLoadData(gfx950 cache object)");
    if ((e = hipModuleLoadData(&o->logprobs, dfq_logprobs_hsaco)) != hipSuccess)
        return hip_error(e, "hipModuleLoadData(gfx950 log-probability object)");
    char name[80];
    static const char* kAttn[3] = {dfq_attn64_hsaco, dfq_attn128_hsaco, dfq_attn256_hsaco};
    for (int d = 0; d < 3; ++d)
        if ((e = hipModuleLoadData(&o->attention[d], kAttn[d])) != hipSuccess)
            return hip_error(e, "hipModuleLoadData(gfx950 attention object)");
    for (int d = 0; d < 3; ++d)
        for (int b = 0; b < 2; ++b)
            for (int g = 0; g < 3 && 32 << g <= 64 << d; ++g)
                for (int t = 0; t < 2; ++t) {
                    CacheKernels& c = o->cache[d][b][g][t];
                    const struct { const char* op; hipFunction_t* fn; } parts[] = {
                        {"append", &c.append}, {"read", &c.read}};
                    for (const auto& part : parts) {
                        snprintf(name, sizeof name, "dfq_cache_%s_d%d_b%d_g%d_%s", part.op,
                                 64 << d, 4 << b, 32 << g, kDt[t]);
                        if ((e = hipModuleGetFunction(part.fn, o->kv, name)) != hipSuccess)
                            return hip_error(e, name);
                    }
                    for (int r = 0; r < attention_tiles(64 << d); ++r) {
                        snprintf(name, sizeof name, "dfq_cache_attention_b%d_g%d_%s_r%d", 4 << b,
                                 32 << g, kDt[t], r + 1);
                        if ((e = hipModuleGetFunction(&c.attention[r], o->attention[d], name)) !=
                            hipSuccess)
                            return hip_error(e, name);
                        if ((e = hipModuleOccupancyMaxActiveBlocksPerMultiprocessor(
                                 &c.resident[r], c.attention[r], DFQ_KV_THREADS, 0)) != hipSuccess)
                            return hip_error(e, name);
                        if (c.resident[r] < 1) return fail(DFQ_ERR_HIP, "%s does not fit", name);
                    }
                    snprintf(name, sizeof name, "dfq_cache_attention_join_g%d_%s", 32 << g, kDt[t]);
                    if ((e = hipModuleGetFunction(&c.join, o->attention[d], name)) != hipSuccess)
                        return hip_error(e, name);
                }
    for (int t = 0; t < 3; ++t) {
        snprintf(name, sizeof name, "dfq_token_logprobs_%s", kDt[t]);
        if ((e = hipModuleGetFunction(&o->logprobs_part[t], o->logprobs, name)) != hipSuccess)
            return hip_error(e, name);
        snprintf(name, sizeof name, "dfq_token_logprobs_join_%s", kDt[t]);
        if ((e = hipModuleGetFunction(&o->logprobs_join[t], o->logprobs, name)) != hipSuccess)
            return hip_error(e, name);
    }
    return DFQ_OK;
}

int dim_index(int dim) { return dim == 64 ? 0 : dim == 128 ? 1 : dim == 256 ? 2 : -1; }
int group_index(int gs) { return gs == 32 ? 0 : gs == 64 ? 1 : gs == 128 ? 2 : -1; }

dfq_status check_format(const dfq_kv_cache* c) {
    if (c->dtype != DFQ_BF16 && c->dtype != DFQ_F16)
        return fail(DFQ_ERR_UNSUPPORTED, "a cache's dtype is bf16 or fp16");
    if (c->bits != 4 && c->bits != 8) return fail(DFQ_ERR_UNSUPPORTED, "bits must be 4 or 8");
    if (dim_index(c->head_dim) < 0)
        return fail(DFQ_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256 (got %d)", c->head_dim);
    if (group_index(c->group_size) < 0 || c->group_size > c->head_dim)
        return fail(DFQ_ERR_UNSUPPORTED,
                    "group size must be 32, 64 or 128 and divide the head (got %d)",
                    c->group_size);
    if (c->slots < 1 || c->heads < 1 || c->capacity < 1)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "slots, heads and capacity must be >= 1");
    if (c->heads > kMostGrid || c->slots > kMostGrid / 2)
        return fail(DFQ_ERR_UNSUPPORTED, "at most %d heads and %d slots", kMostGrid,
                    kMostGrid / 2);
    /* offsets inside one head of one slot are 32 bits in the kernels */
    if ((int64_t)c->capacity * c->head_dim * c->bits / 8 > INT32_MAX)
        return fail(DFQ_ERR_UNSUPPORTED, "one head of one slot must be smaller than 2 GiB");
    return DFQ_OK;
}

dfq_status check_cache(const dfq_kv_cache* c) {
    if (!c) return fail(DFQ_ERR_INVALID_ARGUMENT, "null cache");
    const dfq_status s = check_format(c);
    if (s) return s;
    if (!c->k_codes || !c->k_scales || !c->k_biases || !c->v_codes || !c->v_scales ||
        !c->v_biases)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "null cache array");
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "cache codes must be 16-byte aligned");
    if (!aligned(c->k_scales, 2) || !aligned(c->k_biases, 2) || !aligned(c->v_scales, 2) ||
        !aligned(c->v_biases, 2))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "cache scales and biases must be 2-byte aligned");
    return DFQ_OK;
}

/* Workgroups of an append or read of one sequence: 8 channels a thread, the heads of the same rows
 * side by side, so that they touch the dense side's rows together. */
int64_t row_blocks(const dfq_kv_cache* c, int rows) {
    const int64_t per = DFQ_KV_THREADS * 8 / c->head_dim;
    return (rows + per - 1) / per * c->heads;
}

dfq_status check_span(const dfq_kv_cache* c, int batch, int rows) {
    if (batch < 1 || rows < 1) return fail(DFQ_ERR_INVALID_ARGUMENT, "batch and rows must be >= 1");
    if (batch > c->slots)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "%d sequences in a cache of %d slots", batch,
                    c->slots);
    if (row_blocks(c, rows) > INT32_MAX) return fail(DFQ_ERR_UNSUPPORTED, "grid too large");
    return DFQ_OK;
}

const CacheKernels& kernels_of(const VerifyOps* ops, const dfq_kv_cache* c) {
    return ops->cache[dim_index(c->head_dim)][c->bits == 8][group_index(c->group_size)]
                     [c->dtype == DFQ_F16];
}

KvArrays arrays_of(const dfq_kv_cache* c, bool v) {
    return v ? KvArrays{c->v_codes, (uint16_t*)c->v_scales, (uint16_t*)c->v_biases}
             : KvArrays{c->k_codes, (uint16_t*)c->k_scales, (uint16_t*)c->k_biases};
}

/* The sizes of an attention call; *fmt gets the cache that carries the format. */
dfq_status check_attention(const dfq_kv_cache* prefix, int prefix_length,
                           const dfq_kv_cache* cache, int max_length, int batch, int rows,
                           int q_heads, const dfq_kv_cache** fmt) {
    if (batch < 1 || rows < 1) return fail(DFQ_ERR_INVALID_ARGUMENT, "batch and rows must be >= 1");
    if (rows > DFQ_MAXIMUM_ROWS)
        return fail(DFQ_ERR_UNSUPPORTED, "a block has at most %d rows (got %d)", DFQ_MAXIMUM_ROWS,
                    rows);
    if (batch > kMostGrid) return fail(DFQ_ERR_UNSUPPORTED, "at most %d sequences", kMostGrid);
    if (prefix_length < 0 || max_length < 0)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "negative length");
    if (!prefix && prefix_length) return fail(DFQ_ERR_INVALID_ARGUMENT, "null prefix");
    if (!cache && max_length) return fail(DFQ_ERR_INVALID_ARGUMENT, "null cache");
    if (!prefix && !cache) return fail(DFQ_ERR_INVALID_ARGUMENT, "neither a prefix nor a cache");
    dfq_status s;
    if (prefix) {
        if ((s = check_format(prefix))) return s;
        if (prefix_length > prefix->capacity)
            return fail(DFQ_ERR_INVALID_ARGUMENT, "prefix_length %d is past the capacity %d",
                        prefix_length, prefix->capacity);
    }
    if (cache) {
        if ((s = check_format(cache)) || (s = check_span(cache, batch, rows))) return s;
        if (max_length > cache->capacity)
            return fail(DFQ_ERR_INVALID_ARGUMENT, "max_length %d is past the capacity %d",
                        max_length, cache->capacity);
    }
    if (prefix && cache &&
        (prefix->heads != cache->heads || prefix->head_dim != cache->head_dim ||
         prefix->bits != cache->bits || prefix->group_size != cache->group_size ||
         prefix->dtype != cache->dtype))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "the prefix and the cache differ in format");
    *fmt = cache ? cache : prefix;
    if (q_heads < 1 || q_heads % (*fmt)->heads || q_heads > kMostGrid)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "q_heads %d is not a multiple of the %d heads",
                    q_heads, (*fmt)->heads);
    return DFQ_OK;
}

/* How an attention call is cut: row blocks of tiles * 16 rows, and ranges of tokens. */
struct AttentionPlan {
    int tiles = 1;      /* most row tiles of a block */
    int prefix_splits = 0, prefix_blocks = 0, own_splits = 0, own_blocks = 0;
    int64_t rows = 0;   /* part rows of a slot: heads * batch * rows * group */
    size_t ml_bytes = 0, bytes = 0;
    int64_t groups(int heads, int batch) const {
        return (int64_t)heads * ((int64_t)prefix_splits * prefix_blocks +
                                 (int64_t)batch * own_splits * own_blocks);
    }
};

/* Tokens that a workgroup takes in one round, 32 a wave. */
constexpr int kRoundTokens = DFQ_KV_THREADS / 2;
/* The plan's model of time, in rounds of a workgroup that has a CU to itself: what a workgroup
 * costs besides its rounds (staging the queries, joining its waves); what each workgroup more on
 * a CU adds to a round of all (they wait for memory, then for issue); what two tiles cost against
 * one; and what one more range costs the join.  Over the plans of sixteen shapes (heads of 64, 128
 * and 256, 1..32 sequences, own caches and shared prefixes, groups of 32, 64 and 128) the one that
 * these numbers choose is within 2 % of the fastest, mostly the fastest itself. */
constexpr double kFixedRounds = 1.5, kAnother = 0.45, kTwoTiles = 1.7, kRangeRounds = 0.02;
/* And the join itself, a launch that a single range does without; a round of heads of 256 is twice
 * one of 128.  Device time of 8 rows of 4 sequences (a caller that launches one call after the other
 * saves 2.5 us of its own besides), one range / 128 tokens a range:
 *   heads of 128: 129 tokens 8.6 / 10.4 us, 512 11.2 / 10.7;  64: 7.2 / 8.8, 8.9 / 9.2;
 *   heads of 256: 12.6 / 14.0, 17.2 / 15.2. */
double join_rounds(int dim) { return dim > 128 ? 1.5 : 3.0; }

/* The workgroups of `blocks` row blocks over `rounds` rounds in ranges of at most `each`, as even
 * as they come, by themselves: how long, and how much. */
struct Share {
    double time = 0, work = 0;
    int64_t groups = 0;
    int ranges = 0;
    double longest = 0;   /* a workgroup */
};
struct Card {
    int cus, resident;
    double cost(int64_t groups) const {
        const int64_t per = std::min<int64_t>(resident, (groups + cus - 1) / cus);
        return 1.0 + kAnother * (per - 1);
    }
    Share share(int64_t blocks, int rounds, int each) const {
        Share s;
        if (!rounds) return s;
        s.ranges = (rounds + each - 1) / each;
        each = (rounds + s.ranges - 1) / s.ranges;
        const int whole = rounds / each, last = rounds - whole * each;
        const int64_t room = (int64_t)cus * resident, full = blocks * whole;
        const int64_t passes = full / room, rest = full - passes * room;
        s.longest = each + kFixedRounds;
        s.groups = blocks * s.ranges;
        s.work = (double)blocks * (rounds + s.ranges * kFixedRounds);
        s.time = passes * s.longest * cost(room);
        if (rest && last && rest + blocks <= room)   /* the short ones beside the others */
            s.time += (last + kFixedRounds) * cost(rest + blocks) + (each - last) * cost(rest);
        else if (rest)
            s.time += s.longest * cost(rest);
        if (last && (!rest || rest + blocks > room))   /* behind the first that end */
            s.time += 0.5 * (last + kFixedRounds);
        return s;
    }
};

AttentionPlan plan_attention(int cus, const CacheKernels& kernels, const dfq_kv_cache* fmt,
                             int prefix_length, int max_length, int batch, int rows, int q_heads) {
    AttentionPlan a;
    const int group = q_heads / fmt->heads;
    const int64_t own_rows = (int64_t)rows * group, all_rows = own_rows * batch;
    a.rows = fmt->heads * all_rows;
    const int prefix_rounds = (prefix_length + kRoundTokens - 1) / kRoundTokens;
    const int own_rounds = (max_length + kRoundTokens - 1) / kRoundTokens;
    const int longest = std::max(prefix_rounds, own_rounds);
    const int most = std::min<int64_t>(attention_tiles(fmt->head_dim),
                                       ((prefix_length ? all_rows : own_rows) + 15) / 16);
    double best = 0;
    for (int tiles = 1; tiles <= most; ++tiles) {
        const Card card = {cus, kernels.resident[tiles - 1]};
        const int64_t pb = (all_rows + 16 * tiles - 1) / (16 * tiles);
        const int64_t ob = (own_rows + 16 * tiles - 1) / (16 * tiles);
        const int64_t pn = fmt->heads * pb, on = fmt->heads * ob * batch;
        const double round = tiles == 1 ? 1.0 : kTwoTiles;
        const double all = (double)pn * prefix_rounds + (double)on * own_rounds;
        const int64_t room = (int64_t)card.cus * card.resident;
        /* one range, and ranges that fill every CU with 1, 2, .. workgroups, in one pass and in
         * some */
        for (int fill = 0; fill <= card.resident + 3 && longest; ++fill) {
            const int more = fill - card.resident;
            const int per = more <= 0 ? fill : card.resident * (1 + more);
            const double even =
                fill ? std::floor(all / ((double)card.cus * per)) : (double)longest;
            /* rounded down and up; own ranges of the prefix's length, and of half of it */
            for (int way = 0; way < (prefix_rounds && own_rounds ? 4 : 2); ++way) {
                const int each = (int)std::min<double>(longest, std::max(1.0, even + way % 2));
                const Share p = card.share(pn, prefix_rounds, each);
                const Share o = card.share(on, own_rounds, way < 2 ? each : (each + 1) / 2);
                double t = p.time + o.time;
                if (p.groups && o.groups) {
                    /* the prefix's workgroups come first, and the others fill what they leave */
                    const int64_t n = p.groups + o.groups;
                    const int64_t busy =
                        std::min<int64_t>(card.resident, (n + card.cus - 1) / card.cus);
                    const double work = (p.work + o.work) / (card.cus * busy) * card.cost(n);
                    t = std::max(p.time, n <= room ? std::max(o.longest * card.cost(n), work)
                                                   : work + 0.3 * o.longest);
                }
                t = t * round + kRangeRounds * (p.ranges + o.ranges);
                if (p.ranges + o.ranges > 1) t += join_rounds(fmt->head_dim);
                if (best == 0 || t < best) {
                    best = t;
                    a.tiles = tiles;
                    a.prefix_splits = p.ranges;
                    a.own_splits = o.ranges;
                    a.prefix_blocks = (int)pb;
                    a.own_blocks = (int)ob;
                }
            }
        }
    }
    const size_t slots = (size_t)a.prefix_splits + a.own_splits;
    if (slots == 1) return a;
    a.ml_bytes = (slots * a.rows * 8 + 255) & ~(size_t)255;
    a.bytes = a.ml_bytes + slots * a.rows * fmt->head_dim * 4;
    return a;
}

}  // namespace

extern "C" {

dfq_status dfq_cache_append(dfq_ctx* ctx, const dfq_kv_cache* cache, const void* k, const void* v,
                            int64_t row_stride, int batch, int rows, int start,
                            const int32_t* starts, void* stream) {
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    dfq_status s = check_cache(cache);
    if (s || (s = check_span(cache, batch, rows))) return s;
    if (!k || !v) return fail(DFQ_ERR_INVALID_ARGUMENT, "null k or v");
    if (!aligned(k, 2) || !aligned(v, 2) || !aligned(starts, 4))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned k, v or starts");
    if (row_stride < (int64_t)cache->heads * cache->head_dim)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "row_stride is smaller than a row");
    KvAppendParams p{{arrays_of(cache, false), arrays_of(cache, true)},
                     {(const uint16_t*)k, (const uint16_t*)v}, starts, row_stride, start, rows,
                     cache->heads, cache->capacity};
    const VerifyOps* ops;
    if ((s = ops_of(ctx, &ops))) return s;
    DeviceScope scope(ctx);
    void* args[] = {&p};
    const hipError_t e = hipModuleLaunchKernel(
        kernels_of(ops, cache).append, (unsigned)row_blocks(cache, rows), 1, (unsigned)batch,
        DFQ_KV_THREADS, 1, 1, 0, (hipStream_t)stream, args, nullptr);
    return e == hipSuccess ? DFQ_OK : hip_error(e, "launch dfq_cache_append");
}

dfq_status dfq_cache_read(dfq_ctx* ctx, const dfq_kv_cache* cache, void* k, void* v,
                          dfq_dtype dtype, int batch, int rows, int start, const int32_t* starts,
                          void* stream) {
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    dfq_status s = check_cache(cache);
    if (s || (s = check_span(cache, batch, rows))) return s;
    if (!k && !v) return fail(DFQ_ERR_INVALID_ARGUMENT, "null k and v");
    if (dtype != cache->dtype && dtype != DFQ_F32)
        return fail(DFQ_ERR_UNSUPPORTED, "values are read in the cache's dtype or fp32");
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(starts, 4))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned k, v or starts");
    KvReadParams p{{arrays_of(cache, false), arrays_of(cache, true)}, {k, v}, starts, start, rows,
                   cache->heads, cache->capacity};
    int dt = (int)dtype;
    const VerifyOps* ops;
    if ((s = ops_of(ctx, &ops))) return s;
    DeviceScope scope(ctx);
    void* args[] = {&p, &dt};
    const hipError_t e = hipModuleLaunchKernel(
        kernels_of(ops, cache).read, (unsigned)row_blocks(cache, rows), 1, 2u * batch,
        DFQ_KV_THREADS, 1, 1, 0, (hipStream_t)stream, args, nullptr);
    return e == hipSuccess ? DFQ_OK : hip_error(e, "launch dfq_cache_read");
}

dfq_status dfq_cache_attention_workspace_bytes(dfq_ctx* ctx, const dfq_kv_cache* prefix,
                                               int prefix_length, const dfq_kv_cache* cache,
                                               int max_length, int batch, int rows, int q_heads,
                                               size_t* bytes) {
    if (!bytes) return fail(DFQ_ERR_INVALID_ARGUMENT, "null bytes");
    *bytes = 0;
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    const dfq_kv_cache* fmt;
    dfq_status s =
        check_attention(prefix, prefix_length, cache, max_length, batch, rows, q_heads, &fmt);
    const VerifyOps* ops;
    if (s || (s = ops_of(ctx, &ops))) return s;
    *bytes = plan_attention(dfq_num_cus(ctx), kernels_of(ops, fmt), fmt, prefix_length, max_length,
                            batch, rows, q_heads)
                 .bytes;
    return DFQ_OK;
}

dfq_status dfq_cache_attention(dfq_ctx* ctx, const dfq_kv_cache* prefix, int prefix_length,
                               const dfq_kv_cache* cache, const int32_t* lengths, int max_length,
                               const uint32_t* tree, const void* q, int64_t q_stride, void* y,
                               float* lse, int batch, int rows, int q_heads, float scale,
                               void* workspace, size_t workspace_bytes, void* stream) {
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    const dfq_kv_cache* fmt;
    dfq_status s =
        check_attention(prefix, prefix_length, cache, max_length, batch, rows, q_heads, &fmt);
    if (s || (prefix && (s = check_cache(prefix))) || (cache && (s = check_cache(cache)))) return s;
    if (!q || !y) return fail(DFQ_ERR_INVALID_ARGUMENT, "null q or y");
    if (!cache && (lengths || tree))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "lengths and tree are of a cache, and it is null");
    if (!aligned(q, 2) || !aligned(y, 16) || !aligned(lse, 4) || !aligned(lengths, 4) ||
        !aligned(tree, 4))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned q, y, lse, lengths or tree");
    if (q_stride < (int64_t)q_heads * fmt->head_dim)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "q_stride is smaller than a row");
    if (!(scale > 0.0f) || !std::isfinite(scale))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
    const VerifyOps* ops;
    if ((s = ops_of(ctx, &ops))) return s;
    const CacheKernels& fn = kernels_of(ops, fmt);
    const AttentionPlan a = plan_attention(dfq_num_cus(ctx), fn, fmt, prefix_length, max_length,
                                           batch, rows, q_heads);
    const int64_t groups = a.groups(fmt->heads, batch);
    const int group = q_heads / fmt->heads;
    if (groups > INT32_MAX || (int64_t)batch * rows * group > INT32_MAX)
        return fail(DFQ_ERR_UNSUPPORTED, "grid too large");
    if (a.bytes && (!workspace || workspace_bytes < a.bytes))
        return fail(DFQ_ERR_WORKSPACE, "workspace of %zu bytes needed (got %zu)", a.bytes,
                    workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    KvAttnParams p{};
    if (prefix)
        for (int i = 0; i < 2; ++i) p.prefix[i] = arrays_of(prefix, i);
    if (cache)
        for (int i = 0; i < 2; ++i) p.own[i] = arrays_of(cache, i);
    p.q = (const uint16_t*)q;
    p.y = (uint16_t*)y;
    p.lse = lse;
    p.lengths = lengths;
    p.tree = tree;
    p.part_ml = (float*)workspace;
    p.part_o = (float*)((char*)workspace + a.ml_bytes);
    p.q_stride = q_stride;
    p.prefix_length = prefix_length;
    p.prefix_capacity = prefix ? prefix->capacity : 0;
    p.own_capacity = cache ? cache->capacity : 0;
    p.max_length = max_length;
    p.batch = batch;
    p.rows = divisor(rows);
    p.heads = divisor(fmt->heads);
    p.group = divisor(group);
    p.prefix_splits = divisor(a.prefix_splits);
    p.prefix_blocks = divisor(a.prefix_blocks);
    p.own_splits = divisor(a.own_splits);
    p.own_blocks = divisor(a.own_blocks);
    p.own_jobs = divisor(a.own_splits * a.own_blocks);
    /* a wave joins up to eight slots with all loads under way: 5120 rows of 4 slots 5.3 us, with a
     * workgroup each 11; past eight the other way about (a call of 40 rows of 17 slots 11.1 us, with
     * a wave each 12.5) */
    p.join_rows = a.prefix_splits + a.own_splits <= 8 ? DFQ_KV_THREADS / 64 : 1;
    p.scale_log2e = scale * 1.44269504088896340736f;
    DeviceScope scope(ctx);
    void* args[] = {&p};
    hipError_t e = hipSuccess;
    if (groups)
        e = hipModuleLaunchKernel(fn.attention[a.tiles - 1], (unsigned)groups, 1, 1,
                                  DFQ_KV_THREADS, 1, 1, 0, (hipStream_t)stream, args, nullptr);
    if (e == hipSuccess && a.prefix_splits + a.own_splits != 1)
        e = hipModuleLaunchKernel(fn.join,
                                  (unsigned)(((int64_t)batch * rows * group + p.join_rows - 1) /
                                             p.join_rows),
                                  (unsigned)fmt->heads, 1, DFQ_KV_THREADS, 1, 1, 0,
                                  (hipStream_t)stream, args, nullptr);
    return e == hipSuccess ? DFQ_OK : hip_error(e, "launch dfq_cache_attention");
}

static dfq_status check_logprobs(int M, int V, int top_k) {
    if (M < 1 || V < 1) return fail(DFQ_ERR_INVALID_ARGUMENT, "M and V must be positive");
    if (V > 0x7fffffff / 2) return fail(DFQ_ERR_UNSUPPORTED, "V too large");
    if (top_k < 0 || top_k > DFQ_TOP_MAX)
        return fail(DFQ_ERR_UNSUPPORTED, "top_k must be 0..%d (got %d)", DFQ_TOP_MAX, top_k);
    return DFQ_OK;
}

/* Workgroups a row: ranges of 1024 logits a wave or more, and no more workgroups than the five a CU
 * that are there at once (registers).  64 rows of 151936 with 20 alternatives 18.5 us, 128 25.7, 300
 * with 5 32.3; for eight a CU 23.0, 29.5 and 37.5, for two 21.9, 28.7 and 44.0.  With ranges of 2048
 * logits a wave 8 rows with 5 take 12.6 us against 12.2. */
static int logprob_splits(int num_cus, int M, int V) {
    const int most = std::max(1, 5 * num_cus / M);
    return std::min({most, (int)(((int64_t)V + 4095) / 4096), 64});
}

/* The keys of the rows' parts, then their sums. */
static size_t logprob_keys_bytes(int M, int splits, int top_k) {
    return ((size_t)M * splits * top_k * 8 + 15) & ~(size_t)15;
}
static size_t logprob_bytes(int M, int splits, int top_k) {
    if (splits == 1) return 0;
    return logprob_keys_bytes(M, splits, top_k) + (size_t)M * splits * 16;
}

dfq_status dfq_token_logprobs_workspace_bytes(dfq_ctx* ctx, int M, int V, int top_k,
                                              size_t* bytes) {
    if (!bytes) return fail(DFQ_ERR_INVALID_ARGUMENT, "null bytes");
    *bytes = 0;
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    const dfq_status s = check_logprobs(M, V, top_k);
    if (s) return s;
    *bytes = logprob_bytes(M, logprob_splits(dfq_num_cus(ctx), M, V), top_k);
    return DFQ_OK;
}

dfq_status dfq_token_logprobs(dfq_ctx* ctx, const void* logits, int64_t row_stride, int M, int V,
                              dfq_dtype dtype, const int32_t* tokens, int top_k, float* logprobs,
                              float* entropy, int32_t* top_tokens, float* top_logprobs,
                              void* workspace, size_t workspace_bytes, void* stream) {
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    if (!logits) return fail(DFQ_ERR_INVALID_ARGUMENT, "null logits");
    dfq_status s = check_logprobs(M, V, top_k);
    if (s) return s;
    if (dtype != DFQ_BF16 && dtype != DFQ_F16 && dtype != DFQ_F32)
        return fail(DFQ_ERR_UNSUPPORTED, "logits are bf16, fp16 or fp32");
    if (row_stride < V) return fail(DFQ_ERR_INVALID_ARGUMENT, "row_stride is smaller than a row");
    if (tokens && !logprobs) return fail(DFQ_ERR_INVALID_ARGUMENT, "null logprobs");
    if (top_k && (!top_tokens || !top_logprobs))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "null top_tokens or top_logprobs");
    if (!tokens && !entropy && !top_k)
        return fail(DFQ_ERR_INVALID_ARGUMENT, "nothing is asked for");
    if (!aligned(logits, dtype == DFQ_F32 ? 4 : 2) || !aligned(tokens, 4) ||
        !aligned(logprobs, 4) || !aligned(entropy, 4) || !aligned(top_tokens, 4) ||
        !aligned(top_logprobs, 4))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned buffer");
    const int splits = logprob_splits(dfq_num_cus(ctx), M, V);
    const size_t need = logprob_bytes(M, splits, top_k);
    if (need && (!workspace || workspace_bytes < need))
        return fail(DFQ_ERR_WORKSPACE, "workspace of %zu bytes needed (got %zu)", need,
                    workspace ? workspace_bytes : (size_t)0);
    if (!aligned(workspace, 16))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    if ((int64_t)M * splits > INT32_MAX) return fail(DFQ_ERR_UNSUPPORTED, "grid too large");
    LogprobParams p{logits, tokens, logprobs, entropy, top_tokens, top_logprobs,
                    (uint64_t*)workspace,
                    (float*)((char*)workspace + logprob_keys_bytes(M, splits, top_k)), row_stride,
                    M, V, top_k, splits};
    const VerifyOps* ops;
    if ((s = ops_of(ctx, &ops))) return s;
    DeviceScope scope(ctx);
    void* args[] = {&p};
    hipError_t e = hipModuleLaunchKernel(ops->logprobs_part[(int)dtype], (unsigned)M * splits, 1,
                                         1, DFQ_KV_THREADS, 1, 1, 0, (hipStream_t)stream, args,
                                         nullptr);
    if (e == hipSuccess && splits > 1)
        e = hipModuleLaunchKernel(ops->logprobs_join[(int)dtype], (unsigned)M, 1, 1, 64, 1, 1, 0,
                                  (hipStream_t)stream, args, nullptr);
    return e == hipSuccess ? DFQ_OK : hip_error(e, "launch dfq_token_logprobs");
}

}  // extern "C"
