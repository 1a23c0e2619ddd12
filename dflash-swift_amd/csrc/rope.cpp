/*
 * rope.cpp -- the C ABI of the rotary positions: frequency tables (host only), argument checks and
 * launches of rope.hip.
 */
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "verify_ops.h"

#ifndef DFQ_ROPE_HSACO_PATH
#error "DFQ_ROPE_HSACO_PATH must name the gfx950 code object to embed"
#endif
DFQ_EMBED(dfq_rope_hsaco, DFQ_ROPE_HSACO_PATH)

using namespace dfq;

namespace {

struct RotationOps : LoadedOps {
    static constexpr OpsGroup kGroup = kRotationOps;
    hipModule_t module = nullptr;
    /* [alone/with norms/with norms of a small eps][halves/pairs/any][bf16/f16/f32] */
    hipFunction_t rotate[3][3][3] = {};
    dfq_status resolve() {
        static const char* kDt[3] = {"bf16", "f16", "f32"};
        static const char* kWay[3] = {"halves", "pairs", "any"};
        static const char* kOp[3] = {"rope", "norm_rope", "norm_small_rope"};
        hipError_t e = hipModuleLoadData(&module, dfq_rope_hsaco);
        if (e != hipSuccess) return hip_error(e, "hipModuleLoadData(gfx950 rotation object)");
        char name[80];
        for (int n = 0; n < 3; ++n)
            for (int w = 0; w < 3; ++w)
                for (int t = 0; t < 3; ++t) {
                    snprintf(name, sizeof name, "dfq_%s_%s_%s", kOp[n], kWay[w], kDt[t]);
                    if ((e = hipModuleGetFunction(&rotate[n][w][t], module, name)) != hipSuccess)
                        return hip_error(e, name);
                }
        return DFQ_OK;
    }
    ~RotationOps() override {
        if (module) (void)hipModuleUnload(module);
    }
};

constexpr double kTurn = 6.28318530717958647692528676655900577;

/* f / (2 pi) mod 1 in units of 2^-64, to the nearest: f = m 2^e, m a whole number of 53 bits, times
 * 1 / (2 pi) in units of 2^-256, whose rounding is less than 2^-129 turns of any |f| < 2^127.  (A
 * quotient of 64 bits, its whole turns dropped afterwards, loses as many bits as they have.) */
uint64_t turn_of(double f) {
    static constexpr uint64_t kOverTurn[4] = {0x7f9458eaf7aef158ull, 0x36d8a5664f10e410ull,
                                              0x7f09d5f47d4d3770ull, 0x28be60db9391054aull};
    int e;
    const uint64_t m = (uint64_t)std::ldexp(std::frexp(std::fabs(f), &e), 53);
    uint64_t product[5], carry = 0;   /* in units of 2^(e - 309) turns */
    for (int i = 0; i < 4; ++i) {
        const unsigned __int128 v = (unsigned __int128)m * kOverTurn[i] + carry;
        product[i] = (uint64_t)v;
        carry = (uint64_t)(v >> 64);
    }
    product[4] = carry;
    const auto bit = [&](int at) { return at < 0 || at > 319 ? 0 : product[at / 64] >> at % 64 & 1; };
    const int from = 245 - e;         /* the bit of 2^-64 turns */
    uint64_t turn = 0;
    for (int i = 63; i >= 0; --i) turn = turn << 1 | bit(from + i);
    turn += bit(from - 1);
    return f < 0 ? 0 - turn : turn;
}

bool good(double v) { return v > 0 && std::isfinite(v); }

dfq_status check_heads(const dfq_heads* t, const char* name, dfq_dtype dtype) {
    if (!t->in || !t->out) return fail(DFQ_ERR_INVALID_ARGUMENT, "null %s", name);
    if (!aligned(t->in, dtype_size(dtype)) || !aligned(t->out, dtype_size(dtype)))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned %s", name);
    if (t->heads < 1) return fail(DFQ_ERR_INVALID_ARGUMENT, "%s has no heads", name);
    if (t->heads > kMostGrid)
        return fail(DFQ_ERR_UNSUPPORTED, "at most %d heads (got %d)", kMostGrid, t->heads);
    return DFQ_OK;
}

RopeTensor tensor_of(const dfq_heads* t, const void* weight) {
    return {t->in, t->out, weight, t->in_batch, t->in_row, t->in_head,
            t->out_batch, t->out_row, t->out_head, t->heads, divisor(t->heads)};
}

struct Norms {
    const void* q_weight;
    const void* k_weight;
    dfq_dtype weight_dtype;
    float eps, offset;
};

/* Both entry points; norms is NULL for the rotation alone. */
dfq_status rotate(dfq_ctx* ctx, const dfq_rope_table* rope, const dfq_heads* q, const dfq_heads* k,
                  const Norms* norms, int head_dim, dfq_dtype dtype, int batch, int rows, int start,
                  const int32_t* starts, const int32_t* positions, int inverse, void* stream,
                  const char* what) {
    if (!ctx) return fail(DFQ_ERR_INVALID_ARGUMENT, "null context");
    if (!q) return fail(DFQ_ERR_INVALID_ARGUMENT, "null q");
    if (dtype != DFQ_BF16 && dtype != DFQ_F16 && dtype != DFQ_F32)
        return fail(DFQ_ERR_UNSUPPORTED, "heads are bf16, fp16 or fp32");
    if (head_dim < 2 || head_dim > DFQ_ROPE_DIM || head_dim % 2)
        return fail(DFQ_ERR_UNSUPPORTED, "head_dim must be even and at most %d (got %d)",
                    DFQ_ROPE_DIM, head_dim);
    if (batch < 1 || rows < 1) return fail(DFQ_ERR_INVALID_ARGUMENT, "batch and rows must be >= 1");
    if (!rope && !norms) return fail(DFQ_ERR_INVALID_ARGUMENT, "null rope table");
    if (rope) {
        if (!rope->turns || !aligned(rope->turns, 8))
            return fail(DFQ_ERR_INVALID_ARGUMENT, "null or misaligned turns");
        if (rope->rotary_dim < 2 || rope->rotary_dim % 2 || rope->rotary_dim > head_dim)
            return fail(DFQ_ERR_UNSUPPORTED, "rotary_dim must be even and at most the head's %d "
                        "(got %d)", head_dim, rope->rotary_dim);
        if (!std::isfinite(rope->amplitude))
            return fail(DFQ_ERR_INVALID_ARGUMENT, "amplitude must be finite");
    }
    dfq_status s = check_heads(q, "q", dtype);
    if (s || (k && (s = check_heads(k, "k", dtype)))) return s;
    if (!aligned(starts, 4) || !aligned(positions, 4))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned starts or positions");
    if (positions && (starts || start))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "positions take the place of start and starts");
    RopeParams p{};
    p.t[0] = tensor_of(q, norms ? norms->q_weight : nullptr);
    if (k) p.t[1] = tensor_of(k, norms ? norms->k_weight : nullptr);
    if (norms) {
        if (norms->weight_dtype != dtype && norms->weight_dtype != DFQ_F32)
            return fail(DFQ_ERR_UNSUPPORTED, "weights are in the heads' dtype or fp32");
        const size_t a = dtype_size(norms->weight_dtype);
        if (!aligned(norms->q_weight, a) || !aligned(norms->k_weight, a))
            return fail(DFQ_ERR_INVALID_ARGUMENT, "misaligned weights");
        if (!(norms->eps >= 0.0f) || !std::isfinite(norms->eps) || !std::isfinite(norms->offset))
            return fail(DFQ_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0, the offset finite");
        p.weight_f32 = norms->weight_dtype == DFQ_F32;
        p.eps = norms->eps;
        p.offset = norms->offset;
    }
    const int64_t all = (int64_t)q->heads + (k ? k->heads : 0), tokens = (int64_t)batch * rows;
    if (tokens > INT32_MAX / all)
        return fail(DFQ_ERR_UNSUPPORTED, "grid too large");
    p.turns = rope ? rope->turns : nullptr;
    p.pairs = rope ? rope->rotary_dim / 2 : 0;
    p.amplitude = rope ? rope->amplitude : 1.0f;
    p.interleaved = rope && rope->interleaved;
    p.starts = starts;
    p.positions = positions;
    p.start = start;
    p.inverse = inverse != 0;
    p.tokens = (int)tokens;
    p.dim = head_dim;
    p.rows = divisor(rows);
    /* Chunks of 8 channels hold both channels of their pairs where a head is 16 n wide and, with
     * pairs half the rotated width apart, that half is a multiple of 8. */
    const bool chunks = head_dim % 16 == 0 && (p.interleaved || p.pairs % 8 == 0);
    const int way = chunks ? (p.interleaved ? 1 : 0) : 2;
    p.lanes = 64;
    if (chunks)
        for (p.lanes = 1; p.lanes * 16 < head_dim; p.lanes *= 2) {}
    /* Heads a lane, whose angles are found once: as many as leave every SIMD two waves, up to 16
     * (one in rotate_any). */
    const int64_t waves = tokens * all * p.lanes / 64, cus = std::max(1, dfq_num_cus(ctx));
    const int each = chunks ? (int)std::clamp<int64_t>(waves / (8 * cus), 1, 16) : 1;
    const int64_t per = DFQ_KV_THREADS / p.lanes;
    const auto groups = [&](RopeTensor& t) {
        t.slots = divisor((t.heads + each - 1) / each);
        return (tokens * t.slots.by + per - 1) / per;
    };
    const int64_t q_groups = groups(p.t[0]), k_groups = k ? groups(p.t[1]) : 0;
    if (q_groups + k_groups > kMostGroups) return fail(DFQ_ERR_UNSUPPORTED, "grid too large");
    p.q_groups = (int)q_groups;
    const RotationOps* ops;
    if ((s = ops_of(ctx, &ops))) return s;
    DeviceScope scope(ctx);
    void* args[] = {&p};
    const int op = !norms ? 0 : norms->eps < DFQ_NORM_SMALL ? 2 : 1;
    const hipError_t e = hipModuleLaunchKernel(
        ops->rotate[op][way][(int)dtype], (unsigned)(q_groups + k_groups), 1, 1, DFQ_KV_THREADS,
        1, 1, 0, (hipStream_t)stream, args, nullptr);
    return e == hipSuccess ? DFQ_OK : hip_error(e, what);
}

}  // namespace

extern "C" {

dfq_status dfq_rope_frequencies(const dfq_rope_desc* d, double* frequencies, float* amplitude) {
    if (!d || !frequencies) return fail(DFQ_ERR_INVALID_ARGUMENT, "null argument");
    const int R = d->rotary_dim, n = R / 2;
    if (R < 2 || R % 2 || R > DFQ_ROPE_DIM)
        return fail(DFQ_ERR_UNSUPPORTED, "rotary_dim must be even and at most %d (got %d)",
                    DFQ_ROPE_DIM, R);
    if (!(d->base > 1.0) || !std::isfinite(d->base))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "base must be finite and above 1");
    if (d->scaling < DFQ_ROPE_PLAIN || d->scaling > DFQ_ROPE_YARN)
        return fail(DFQ_ERR_UNSUPPORTED, "unknown scaling %d", (int)d->scaling);
    if (d->scaling != DFQ_ROPE_PLAIN && !good(d->factor))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "factor must be positive and finite");
    const bool bands = d->scaling == DFQ_ROPE_BANDS, yarn = d->scaling == DFQ_ROPE_YARN;
    if ((bands || yarn) && !good(d->original_length))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "original_length must be positive and finite");
    if (bands && !(good(d->low_freq_factor) && good(d->high_freq_factor) &&
                   d->low_freq_factor < d->high_freq_factor))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "0 < low_freq_factor < high_freq_factor");
    if (yarn && !(good(d->beta_fast) && good(d->beta_slow) && d->beta_slow < d->beta_fast))
        return fail(DFQ_ERR_INVALID_ARGUMENT, "0 < beta_slow < beta_fast");
    double base = d->base;
    if (d->scaling == DFQ_ROPE_NTK) base *= std::pow(d->factor, (double)R / (R > 2 ? R - 2 : 1));
    double low = 0, high = 0;
    if (yarn) {
        /* the pair that turns `beta` times over the original length */
        const auto edge = [&](double beta) {
            return R * std::log(d->original_length / (beta * kTurn)) / (2 * std::log(base));
        };
        low = std::fmax(std::floor(edge(d->beta_fast)), 0.0);
        high = std::fmin(std::ceil(edge(d->beta_slow)), R - 1.0);
    }
    for (int i = 0; i < n; ++i) {
        const double f = std::pow(base, -2.0 * i / R);
        double keep = 1.0;   /* of the frequency; the rest is divided by the factor */
        if (d->scaling == DFQ_ROPE_LINEAR) keep = 0.0;
        if (bands)
            keep = (d->original_length * f / kTurn - d->low_freq_factor) /
                   (d->high_freq_factor - d->low_freq_factor);
        if (yarn) keep = 1.0 - (i - low) / std::fmax(high - low, 0.001);
        keep = std::fmin(std::fmax(keep, 0.0), 1.0);
        frequencies[i] = keep == 1.0 ? f : keep * f + (1.0 - keep) * f / d->factor;
    }
    if (amplitude)
        *amplitude = yarn && d->factor > 1.0 ? (float)(0.1 * std::log(d->factor) + 1.0) : 1.0f;
    return DFQ_OK;
}

dfq_status dfq_rope_turns(const double* frequencies, int count, uint64_t* turns) {
    if (!frequencies || !turns) return fail(DFQ_ERR_INVALID_ARGUMENT, "null argument");
    if (count < 1) return fail(DFQ_ERR_INVALID_ARGUMENT, "count must be >= 1");
    for (int i = 0; i < count; ++i) {
        if (!(std::fabs(frequencies[i]) < 0x1p127))
            return fail(DFQ_ERR_INVALID_ARGUMENT, "frequency %d is not under 2^127", i);
        turns[i] = turn_of(frequencies[i]);
    }
    return DFQ_OK;
}

dfq_status dfq_rope(dfq_ctx* ctx, const dfq_rope_table* rope, const dfq_heads* q,
                    const dfq_heads* k, int head_dim, dfq_dtype dtype, int batch, int rows,
                    int start, const int32_t* starts, const int32_t* positions, int inverse,
                    void* stream) {
    return rotate(ctx, rope, q, k, nullptr, head_dim, dtype, batch, rows, start, starts, positions,
                  inverse, stream, "launch dfq_rope");
}

dfq_status dfq_qk_norm_rope(dfq_ctx* ctx, const dfq_rope_table* rope, const dfq_heads* q,
                            const dfq_heads* k, const void* q_weight, const void* k_weight,
                            dfq_dtype weight_dtype, float eps, float weight_offset, int head_dim,
                            dfq_dtype dtype, int batch, int rows, int start, const int32_t* starts,
                            const int32_t* positions, void* stream) {
    const Norms norms = {q_weight, k_weight, weight_dtype, eps, weight_offset};
    return rotate(ctx, rope, q, k, &norms, head_dim, dtype, batch, rows, start, starts, positions, 0,
                  stream, "launch dfq_qk_norm_rope");
}

}  // extern "C"
