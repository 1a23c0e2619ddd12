/*
 * sample_accept.hip -- gfx950 kernels that verify drafted tokens against the target's probabilities
 * from given random numbers, and draw the token behind them.
 *
 * With p = softmax(logits / T) of the target's rows and q that of the draft's (or the draft alone,
 * q(d) = 1, where there are no draft logits), draft i is accepted where u_i q_i(d) < p_i(d).  At
 * the first that is not, the token is drawn from max(p - q, 0), behind the last of them from p: the
 * first t whose running sum passes u times the whole.  That keeps the tokens distributed as p.  A
 * temperature of 0 stands for the largest logit alone (the first of equal ones).
 *
 * Tokens and counts are whole numbers that a sum's last bits decide, and come out as 64-bit
 * arithmetic has them (exponentials to 8e-13): draws sum and search in 64 bits, and a draft whose
 * u q is as near to p as fp32 sums may be wrong is decided again from 64-bit ones.  Other drafts
 * need no more than fp32, in which a logit costs 8 instructions against 20: all rows of 64 sequences
 * of seven drafts of 151936 tokens in 64 bits took 93 us for 43.
 *
 * An fp32 sum is off by less than (7/4 log2 V + 20) 2^-24 of itself.  An exponent a of 2 has three
 * roundings (rate, difference, product) of up to 2^-24 |a| each, which change its power by
 * 3 ln 2 |a| 2^-24, and so the sum by the mean of that over the row's mass.  The mean of |a| is largest
 * where all tokens but the largest are alike, W((V-1)/e) / ln 2 with Lambert's W: its 3 W((V-1)/e) is
 * below 7/4 log2 V for any V up to 2^30 (26.3 for 30.1 at 151936 tokens, 50.9 for 52.5 at the most).
 * 13 sums in a row and the last bits of three exponentials (a token's, and the factors that join ranges)
 * are 19 more.
 *
 * The first launch reads all rows once: a wave takes a range of one row in registers, finds its
 * largest logit and the sum of e^((x - largest) / T).  In the second each workgroup joins its
 * sequence's ranges and decides its drafts (alike in all of them, so that nothing has to be waited
 * for), then weighs its part of the row that is drawn from; the last to come finds the token.
 * A draw from p - q needs no third launch either, though its terms are known only when both rows
 * have been summed: nearly all tokens' signs are, from the fp32 sums (from_rest).
 *
 * 64 sequences of seven sampled drafts of 151936 tokens in bf16: 73 us a call where calls follow each
 * other in a graph.  Launches traced one by one, the sums take 43.8 (254 MB, 5.8 TB/s) and the draws 31,
 * of which vector instructions are some 18 and the rest what the launch's start, its decisions and its
 * last workgroup take.  16 sequences 29.5 us, one block of seven certain drafts 12.5, 33 plain draws
 * from 50257 logits in fp32 13.9.
 */
#include "logit_piece.h"

namespace {

constexpr int kWaves = DFQ_KV_THREADS / 64;
constexpr double kLog2e = 1.44269504088896340736, kLn2 = 0.693147180559945309417;
constexpr int kNone = 0x7fffffff;

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

/* 2^f for |f| <= 1/2: the polynomial of degree 8 whose largest relative error, 7.8e-13, is least
 * (its nine alternating extremes found by exchange). */
__device__ __forceinline__ double power_of_part(double f) {
    double s = 0x1.61afcebc3eb7bp-20;
    s = fma(f, s, 0x1.00dad25030da9p-16);
    s = fma(f, s, 0x1.430acca345de3p-13);
    s = fma(f, s, 0x1.5d87483855d3ep-10);
    s = fma(f, s, 0x1.3b2ab5c52926cp-7);
    s = fma(f, s, 0x1.c6b08dd46d38ep-5);
    s = fma(f, s, 0x1.ebfbdff9319e1p-3);
    s = fma(f, s, 0x1.62e42fef8615ep-1);
    return fma(f, s, 0x1.ffffffffff7a3p-1);
}

constexpr double kWhole = 6755399441055744.0;   /* 1.5 2^52: sums with it are whole numbers */
/* Powers stop at 2^-1022, which stands for all that is less; what weighs no more than this is 0. */
constexpr double kNothing = 0x1p-1000;

/* 2^(d rate) for d <= 0, down to 2^-1022; `least` is -1022 / rate. */
__device__ __forceinline__ double power(double d, double rate, double least) {
    d = fmax(d, least);
    const double t = fma(d, rate, kWhole);
    const double v = power_of_part(fma(d, rate, kWhole - t));
    u32x2_t w = __builtin_bit_cast(u32x2_t, v);
    w[1] += __builtin_bit_cast(u32x2_t, t)[0] << 20;
    return __builtin_bit_cast(double, w);
}

__device__ __forceinline__ double rate_of(float t) { return kLog2e / t; }
/* A row's exponentials: of its logits x, 2^((x - top) rate). */
struct Powers {
    double rate, least, top;
    __device__ __forceinline__ Powers(float t, float largest)
        : rate(rate_of(t)), least(-1022.0 * kLn2 * t), top(largest) {}
    __device__ __forceinline__ double operator()(float x) const {
        return power((double)x - top, rate, least);
    }
};
/* The same exponents (x - top) rate in fp32.  Logits may lie further apart than fp32 reaches, which
 * counts where a temperature is as large: there both are taken 2^-8 fold, exactly.  The rate of a
 * temperature under the least normal number has no room in fp32: 2^23 of it go to the difference. */
struct Exponents {
    float fold, lift, rate;
    __device__ __forceinline__ Exponents(float t) {
        const bool large = t > 0x1p100f, small = t < 0x1p-126f;
        fold = large ? 0x1p-8f : 1.0f;
        lift = small ? 0x1p23f : 1.0f;
        rate = (float)(rate_of(t) * (large ? 0x1p8 : small ? 0x1p-23 : 1.0));
    }
    __device__ __forceinline__ float operator()(float x, float top) const {
        return fmaf(x, fold, -(top * fold)) * lift * rate;
    }
};
__device__ __forceinline__ bool is_temperature(float t) {
    return t >= 0.0f && t < __builtin_inff();
}

/* What is alike in all lanes, in scalar registers. */
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}
__device__ __forceinline__ double uniform(double v) {
    u32x2_t w = __builtin_bit_cast(u32x2_t, v);
    w[0] = __builtin_amdgcn_readfirstlane(w[0]);
    w[1] = __builtin_amdgcn_readfirstlane(w[1]);
    return __builtin_bit_cast(double, w);
}

struct Sequence {
    float t, dt;         /* temperatures                        */
    int drafts;          /* that it brings                      */
    bool drafted;        /* q is a softmax of the draft logits  */
};
__device__ __forceinline__ Sequence sequence_of(const AcceptParams& p, int b) {
    Sequence s;
    s.t = p.temperatures ? p.temperatures[b] : p.temperature;
    s.dt = p.draft_temperatures ? p.draft_temperatures[b] : p.draft_temperature;
    s.drafts = p.rows - 1;
    if (p.lengths) {
        const int n = p.lengths[b];
        s.drafts = n < 0 ? 0 : n < s.drafts ? n : s.drafts;
    }
    s.drafted = p.draft_logits && s.dt != 0.0f;
    return s;
}

/* Exchanges over a wave: within rows of 16 lanes by DPP, then across. */
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lanes16_sum(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    return v + dpp_f64<0x140>(v);
}
__device__ __forceinline__ double wave_sum(double v) {
    v = lanes16_sum(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
/* Two sums at once: a's in the lower 32 lanes, b's in the upper. */
__device__ __forceinline__ double wave_sums(double a, double b) {
    const bool upper = threadIdx.x % 64 >= 32;
    const double v = (upper ? b : a) + __shfl_xor(upper ? a : b, 32);
    const double sum = lanes16_sum(v);
    return sum + __shfl_xor(sum, 16);
}
template <typename Op>
__device__ __forceinline__ float wave_of(float v, Op op) {
    const auto bits = [&](uint32_t a, uint32_t b) {
        return __float_as_uint(op(__uint_as_float(a), __uint_as_float(b)));
    };
    v = __uint_as_float(group_of<16>(__float_as_uint(v), bits));
    v = op(v, __shfl_xor(v, 16));
    return op(v, __shfl_xor(v, 32));
}

/* Of two numbers the larger, NaN where one is NaN. */
__device__ __forceinline__ float larger(float a, float b) {
    return __builtin_elementwise_maximum(a, b);
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double waves[kWaves];
    v = wave_sum(v);
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += waves[w];
    __syncthreads();
    return s;
}

__device__ __forceinline__ void block_sums(double& a, double& b) {
    __shared__ double waves[2 * kWaves];
    const double v = wave_sums(a, b);
    if (threadIdx.x % 32 == 0) waves[threadIdx.x / 32] = v;
    __syncthreads();
    a = b = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        a += waves[2 * w];
        b += waves[2 * w + 1];
    }
    __syncthreads();
}

__device__ __forceinline__ double of_lane(double v, int lane) {
    const u32x2_t w = __builtin_bit_cast(u32x2_t, v);
    return __builtin_bit_cast(double, u32x2_t{(uint32_t)__builtin_amdgcn_readlane(w[0], lane),
                                              (uint32_t)__builtin_amdgcn_readlane(w[1], lane)});
}

/* The sum over the threads in front of this one; `all` gets that over all.  The caller has a barrier
 * before the next call. */
__device__ __forceinline__ double block_before(double v, double& all) {
    __shared__ double waves[kWaves];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    /* running sums within rows of 16 lanes, by DPP's shifts, then the rows in front */
    double run = v;
    run += dpp_f64<0x111>(run);
    run += dpp_f64<0x112>(run);
    run += dpp_f64<0x114>(run);
    run += dpp_f64<0x118>(run);
    const double one = of_lane(run, 15), two = one + of_lane(run, 31), three = two + of_lane(run, 47);
    run += lane < 16 ? 0.0 : lane < 32 ? one : lane < 48 ? two : three;
    if (lane == 63) waves[wave] = run;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += waves[w];
        all += waves[w];
    }
    return before + (run - v);
}

/* Of 512 weights, two neighbours a thread: where their running sum, counted from `from`, first
 * passes the goal, or the last that weighs anything, or kNone; `front` gets the sum in front of it.
 * A goal below 0 stands for u times the sum of all, and is set.  The threads' answers meet by
 * ballots (256 lanes' minimum by LDS atomics took 2.5 us). */
struct Search {
    double goal, front;
    int place;
};
__device__ __noinline__ Search search(double a, double b, double from, double goal, double u) {
    __shared__ int firsts[kWaves], lasts[kWaves], place;
    __shared__ double front;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    double all;
    const double run = from + block_before(a + b, all);
    if (goal < 0.0) goal = u * all;
    const bool weighs = a > kNothing || b > kNothing;
    const uint64_t some = __ballot(weighs);
    const uint64_t past = __ballot(weighs && run + (a + b) > goal);
    if (lane == 0) {
        firsts[wave] = past ? (int)__builtin_ctzll(past) : -1;
        lasts[wave] = some ? 63 - (int)__builtin_clzll(some) : -1;
    }
    if (threadIdx.x == 0) place = kNone;
    __syncthreads();
    int first = kNone, last = -1;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (first == kNone && firsts[w] >= 0) first = 64 * w + firsts[w];
        if (lasts[w] >= 0) last = 64 * w + lasts[w];
    }
    if ((int)threadIdx.x == (first != kNone ? first : last)) {
        const bool second = a <= kNothing || (b > kNothing && run + a <= goal);
        place = 2 * (int)threadIdx.x + second;
        front = second ? run + a : run;
    }
    __syncthreads();
    return {goal, front, place};
}

/* The place among n weights where their running sum passes u times their sum (goal < 0), or the
 * goal, counted from `from`: cut into 512 parts until a part is one weight.  A weight is that of
 * (place, what `fetch` reads of it); all threads come to each, those without one to a neighbour's. */
template <typename Fetch, typename Weight>
__device__ __forceinline__ Search find(int n, Fetch fetch, Weight weight, double from, double goal,
                                       double u) {
    int lo = 0;
    for (;;) {
        const int each = (n + 2 * DFQ_KV_THREADS - 1) / (2 * DFQ_KV_THREADS);
        double w[2] = {};
        if (each == 1) {
            /* both loads under way at once: behind a branch each they came one after the other */
            const int i = 2 * (int)threadIdx.x;
            const int at0 = lo + min(i, n - 1), at1 = lo + min(i + 1, n - 1);
            const auto first = fetch(at0), second = fetch(at1);
            w[0] = weight(at0, first);
            w[1] = weight(at1, second);
            w[0] = i < n ? w[0] : 0.0;
            w[1] = i + 1 < n ? w[1] : 0.0;
        } else {
            for (int k = 0; k < 2; ++k) {
                const int64_t begin = (2 * (int64_t)threadIdx.x + k) * each;
                for (int64_t i = begin; i < begin + each; ++i) {
                    const int at = lo + (int)(i < n ? i : n - 1);
                    const double v = weight(at, fetch(at));
                    w[k] += i < n ? v : 0.0;
                }
            }
        }
        Search s = search(w[0], w[1], from, goal, u);
        if (s.place == kNone) return s;
        lo += s.place * each;
        n = min(each, n - s.place * each);
        if (each == 1) {
            s.place = lo;
            return s;
        }
        from = s.front;
        goal = s.goal;
    }
}

/* What is known of a row: its largest logit, and the sum of 2^((x - top) rate) or (T = 0) where
 * it is first. */
struct Row {
    float top;
    int at;
    double sum;
};

/* What is left to draw of a sequence: nothing, or a token from p, from p without its draft, or from
 * max(p - q, 0). */
enum { kDrawNone, kDrawP, kDrawOther, kDrawRest };
struct Draw {
    int mode, row;          /* the target's row, and the place of the token */
    int draft, token;       /* the row's draft; the token of kDrawNone      */
    float p_top, q_top;     /* largest logits of the rows                   */
    double p_sum, q_sum;    /* and their sums, right to fp32's bound        */
};

template <int DT>
struct Accept : LogitPiece<DT> {
    using LogitPiece<DT>::kN, LogitPiece<DT>::load, LogitPiece<DT>::widen;
    static constexpr int kSize = 16 / kN;
    static constexpr int kUnit = 64 * kN;           /* logits of a wave's load          */

    static __device__ __forceinline__ const char* target_row(const AcceptParams& p, int b, int r) {
        return (const char*)p.logits + (b * p.batch_stride + r * p.row_stride) * kSize;
    }
    static __device__ __forceinline__ const char* draft_row(const AcceptParams& p, int b, int r) {
        return (const char*)p.draft_logits +
               (b * p.draft_batch_stride + r * p.draft_row_stride) * kSize;
    }

    /* One range of one row by one wave, kPieces x 16 bytes a lane; its sum in fp32.  Of 2, 3, 4, 6
     * and 8 pieces, 64 sequences of seven drafts took 85, 75, 72, 72 and 73 us, 16 32, 30, 30, 30 and
     * 32 (8 take 108 registers), one block 12.7, 12.1, 12.5, 12.5 and 13.5. */
    static __device__ __forceinline__ void sums(const AcceptParams& p) {
        constexpr int kPieces = DFQ_ACCEPT_PIECES, kRange = kPieces * kUnit;
        const int lane = threadIdx.x % 64;
        const int job = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + threadIdx.x / 64);
        if (job >= p.jobs) return;
        const int row = divided(job, p.ranges), range = job - row * p.ranges.by;
        const int b = divided(row, p.all_rows), r = row - b * p.all_rows.by;
        if (r == 0 && range == 0 && lane == 0) p.arrived[b * DFQ_ACCEPT_APART] = 0;
        const bool draft = r >= p.rows;
        const Sequence q = sequence_of(p, b);
        /* rows behind a sequence's drafts, and draft rows that do not matter */
        if (draft ? r - p.rows >= q.drafts || !q.drafted : r > q.drafts) return;
        const char* at_row = draft ? draft_row(p, b, r - p.rows) : target_row(p, b, r);
        const float t = draft ? q.dt : q.t;
        const int from = range * kRange + lane * kN;
        const bool whole = (range + 1) * kRange <= p.vocab;
        u32x4_t v[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int at = from + i * kUnit;
            v[i] = whole ? *(const u32x4_any*)(at_row + (int64_t)at * kSize)
                         : load(at_row, at, p.vocab);
        }
        AcceptPart part = {-__builtin_inff(), 0};
        if (t == 0.0f) {
            /* the first of the largest, NaN passed over */
            float top = __builtin_nanf("");
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                float x[kN];
                widen(v[i], x);
#pragma unroll
                for (int j = 0; j < kN; ++j) top = fmaxf(top, x[j]);
            }
            top = wave_of(top, [](float a, float c) { return fmaxf(a, c); });
            int at = kNone;
#pragma unroll
            for (int i = kPieces - 1; i >= 0; --i) {
                float x[kN];
                widen(v[i], x);
#pragma unroll
                for (int j = kN - 1; j >= 0; --j)
                    if (x[j] == top && from + i * kUnit + j < p.vocab) at = from + i * kUnit + j;
            }
            for (int d = 1; d < 64; d *= 2) at = min(at, __shfl_xor(at, d));
            part = {top, (uint32_t)at};
        } else {
            float top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                float x[kN];
                widen(v[i], x);
#pragma unroll
                for (int j = 0; j < kN; ++j) top = larger(top, x[j]);
            }
            top = wave_of(top, [](float a, float c) { return larger(a, c); });
            part.top = top;
            if (fabsf(top) < __builtin_inff()) {
                const Exponents exponent(t);
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    float x[kN];
                    widen(v[i], x);
#pragma unroll
                    for (int j = 0; j < kN; ++j)
                        x[j] = __builtin_amdgcn_exp2f(exponent(x[j], top));
                    /* in pairs: fewer roundings in a row */
#pragma unroll
                    for (int d = kN / 2; d; d /= 2)
#pragma unroll
                        for (int j = 0; j < d; ++j) x[j] += x[j + d];
                    sum += x[0];
                }
                part.sum = __float_as_uint(wave_of(sum, [](float a, float c) { return a + c; }));
            }
        }
        if (lane == 0) p.parts[job] = part;
    }

    /* A row's ranges together, by 16 lanes.  NaN, +inf or nothing above -inf leaves a sum that is
     * not positive and finite. */
    static __device__ __forceinline__ Row row_of(const AcceptParams& p, int b, int r, float t) {
        const int lane = threadIdx.x % 16, n = p.ranges.by;
        const int64_t first = ((int64_t)b * p.all_rows.by + r) * n;
        Row row = {-__builtin_inff(), kNone, 0.0};
        const Exponents exponent(t);
        const auto factor = [&](float from, float to) -> double {
            return __builtin_amdgcn_exp2f(exponent(from, to));
        };
        constexpr int kOnce = 4;   /* loads on their way together */
        for (int from = 0; from < n; from += 16 * kOnce) {
            AcceptPart v[kOnce];
            double sums[kOnce];
#pragma unroll
            for (int j = 0; j < kOnce; ++j)
                v[j] = p.parts[first + min(from + 16 * j + lane, n - 1)];
#pragma unroll
            for (int j = 0; j < kOnce; ++j) {
                const bool in = from + 16 * j + lane < n;
                sums[j] = in ? (double)__uint_as_float(v[j].sum) : 0.0;
                v[j].top = in ? v[j].top : -__builtin_inff();
                v[j].sum = in ? v[j].sum : (uint32_t)kNone;
            }
            if (t == 0.0f) {
#pragma unroll
                for (int j = 0; j < kOnce; ++j)
                    if ((int)v[j].sum != kNone && (row.at == kNone || v[j].top > row.top)) {
                        row.top = v[j].top;
                        row.at = (int)v[j].sum;
                    }
                continue;
            }
            float to = row.top;
#pragma unroll
            for (int j = 0; j < kOnce; ++j) to = larger(to, v[j].top);
            if (fabsf(to) < __builtin_inff()) {
                row.sum *= factor(row.top, to);
#pragma unroll
                for (int j = 0; j < kOnce; ++j) row.sum += sums[j] * factor(v[j].top, to);
            }
            row.top = to;
        }
        if (t == 0.0f) {
#pragma unroll
            for (int d = 1; d < 16; d *= 2) {
                const float top = __shfl_xor(row.top, d);
                const int at = __shfl_xor(row.at, d);
                if (at != kNone && (row.at == kNone || top > row.top ||
                                    (top == row.top && at < row.at))) {
                    row.top = top;
                    row.at = at;
                }
            }
            return row;
        }
        const float top = __uint_as_float(
            group_of<16>(__float_as_uint(row.top), [](uint32_t a, uint32_t c) {
                return __float_as_uint(larger(__uint_as_float(a), __uint_as_float(c)));
            }));
        double sum = __builtin_nan("");
        if (fabsf(top) < __builtin_inff())
            sum = row.sum * factor(row.top, top);
        return {top, kNone, lanes16_sum(sum)};
    }

    /* The sum of a whole row in 64 bits, by a workgroup alone. */
    static __device__ __noinline__ double whole_row(const char* row, int vocab, float top,
                                                    float t) {
        const Powers e(t, top);
        constexpr int kOnce = 4, kStep = DFQ_KV_THREADS * kN;   /* loads on their way together */
        double sum = 0.0;
        for (int from = threadIdx.x * kN; from < vocab; from += kOnce * kStep) {
            u32x4_t v[kOnce];
#pragma unroll
            for (int k = 0; k < kOnce; ++k) v[k] = load(row, from + k * kStep, vocab);
#pragma unroll
            for (int k = 0; k < kOnce; ++k) {
                float x[kN];
                widen(v[k], x);
#pragma unroll
                for (int j = 0; j < kN; ++j) sum += e(x[j]);
            }
        }
        return block_sum(sum);
    }

    static __device__ __forceinline__ double counted(double v) { return v > kNothing ? v : 0.0; }

    /* A logit's share of its row. */
    static __device__ __forceinline__ double part_of(float x, float t, float top, double sum) {
        return counted(Powers(t, top)(x)) / sum;
    }

    /* Decides the drafts of sequence b, by a workgroup: 16 lanes join a row, lane i of the last
     * wave looks at draft i.  `writes` stores what is known without a draw. */
    static __device__ __forceinline__ Draw decide(const AcceptParams& p, const Sequence& s,
                                                        int b, bool writes) {
        __shared__ Row rows[2 * 64];
        __shared__ Draw made;
        __shared__ uint64_t again;
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        const bool greedy = s.t == 0.0f;
        /* The last wave decides (with few rows it has none to join), and what it will need of the
         * drafts is on its way meanwhile.  Rows and drafts behind the sequence's own are met too:
         * its length and temperatures need not have come before. */
        const bool decides = wave == kWaves - 1;
        int draft = -1;
        float x = 0.0f, y = 0.0f, u = 0.0f;
        bool known = false;
        if (decides && lane < p.rows - 1) {
            draft = p.drafts[(int64_t)b * (p.rows - 1) + lane];
            u = p.uniforms[(int64_t)b * p.rows + lane];
            known = draft >= 0 && draft < p.vocab;
            if (known) {
                x = load_any(target_row(p, b, lane), DT, draft);
                if (p.draft_logits) y = load_any(draft_row(p, b, lane), DT, draft);
            }
        }
        for (int i = threadIdx.x / 16; i < (int)p.all_rows.by; i += DFQ_KV_THREADS / 16) {
            const Row row = row_of(p, b, i, i < p.rows ? s.t : s.dt);
            if (lane % 16 == 0) rows[i] = row;
        }
        __syncthreads();
        Row row = {0.0f, kNone, 0.0}, other = row;
        bool some = true, taken = false;   /* some: both rows have a distribution */
        double mine = 0.0, theirs = 1.0;
        if (decides) {
            if (lane <= s.drafts) {
                row = rows[lane];
                some = greedy ? row.at != kNone
                              : row.sum > 0.0 && row.sum < __builtin_inf() &&
                                    is_temperature(s.t);
            }
            if (lane < s.drafts) {
                if (s.drafted) {
                    other = rows[p.rows + lane];
                    some = some && other.sum > 0.0 && other.sum < __builtin_inf() &&
                           is_temperature(s.dt);
                }
                known = known && some;
                if (known) {
                    if (greedy) mine = draft == row.at;
                    else mine = part_of(x, s.t, row.top, row.sum);
                    if (s.drafted) theirs = part_of(y, s.dt, other.top, other.sum);
                    taken = u * theirs < mine;
                }
            }
            known = known && lane < s.drafts;
            const uint64_t near =
                __ballot(known && mine > 0.0 && fabs(u * theirs - mine) < p.near * mine);
            if (lane == 0) again = near;
        }
        __syncthreads();
        /* drafts next to the border: one in a hundred thousand or so */
        for (uint64_t near = again; near; near &= near - 1) {
            const int i = __builtin_ctzll(near);
            double p_sum = 0.0, q_sum = 0.0;
            if (!greedy) p_sum = whole_row(target_row(p, b, i), p.vocab, rows[i].top, s.t);
            if (s.drafted)
                q_sum = whole_row(draft_row(p, b, i), p.vocab, rows[p.rows + i].top, s.dt);
            if (decides && lane == i) {
                if (!greedy) mine = part_of(x, s.t, row.top, p_sum);
                if (s.drafted) theirs = part_of(y, s.dt, other.top, q_sum);
                taken = u * theirs < mine;
            }
        }
        if (decides) {
            const uint64_t refused = ~__ballot(taken);
            const int n = __builtin_ctzll(refused);   /* at most 63 drafts: some bit is set */
            if (lane == n) {
                Draw d = {kDrawNone, n, draft, -1, row.top, other.top, row.sum,
                                other.sum};
                if (some && greedy) d.token = row.at;
                else if (some && n == s.drafts) d.mode = kDrawP;
                else if (some) d.mode = s.drafted ? kDrawRest : kDrawOther;
                made = d;
                if (writes) p.accepted[b] = n;
            }
            if (writes) {
                if (p.chances && lane < p.rows - 1) {
                    float chance = 0.0f;
                    if (known) chance = theirs > 0.0 ? (float)fmin(mine / theirs, 1.0) : mine > 0.0;
                    p.chances[(int64_t)b * (p.rows - 1) + lane] = chance;
                }
                if (lane < p.rows && lane != n)
                    p.tokens[(int64_t)b * p.rows + lane] = lane < n ? draft : -1;
            }
        }
        __syncthreads();
        return {uniform(made.mode), uniform(made.row), uniform(made.draft), uniform(made.token),
                uniform(made.p_top), uniform(made.q_top), uniform(made.p_sum),
                uniform(made.q_sum)};
    }

    static __device__ __forceinline__ void put(uint64_t* at, double v) {
        __hip_atomic_store(at, __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    }
    static __device__ __forceinline__ double got(const uint64_t* at) {
        return __builtin_bit_cast(
            double, __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
    /* Whether this is the last of sequence b's workgroups to come.  Sums and count meet in memory,
     * past the caches, by device-scope atomics: a wave's stores have completed before its workgroup
     * counts.  (Fences that write back and drop the L2 instead made 16 sequences' draw take 77
     * us.) */
    static __device__ __forceinline__ bool last(const AcceptParams& p, int b) {
        __shared__ int arrived;
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0)
            arrived = __hip_atomic_fetch_add(&p.arrived[b * DFQ_ACCEPT_APART], 1, __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        return arrived == p.chunks.by - 1;
    }

    /* A token drawn from the exponentials of the target's row, without the one at `without`: waves
     * sum units, and the last of the sequence's workgroups finds it (kNone: nothing weighs), -1 in
     * the others. */
    static __device__ __forceinline__ int from_row(const AcceptParams& p, const char* row,
                                                   const Powers& e, int without, int b, int chunk,
                                                   double u) {
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        uint64_t* sums = p.sums + (int64_t)b * p.sums_apart;
        const auto weight = [&](int i, float x) { return i == without ? 0.0 : e(x); };
        for (int unit = chunk * kWaves + wave; unit < p.units; unit += p.chunks.by * kWaves) {
            const int i = unit * kUnit + lane * kN;
            float x[kN];
            widen(load(row, i, p.vocab), x);
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < kN; ++j) sum += weight(i + j, x[j]);
            sum = wave_sum(sum);
            if (lane == 0) put(&sums[unit], sum);
        }
        if (!last(p, b)) return -1;
        const Search unit = find(p.units, [&](int i) { return got(&sums[i]); },
                                 [](int, double v) { return v; }, 0.0, -1.0, u);
        if (unit.place == kNone) return kNone;
        const int from = unit.place * kUnit;
        const int place = find(min(kUnit, p.vocab - from),
                               [&](int i) { return load_any(row, DT, from + i); },
                               [&](int i, float x) { return weight(from + i, x); },
                               unit.front, unit.goal, u).place;
        if (place != kNone) return from + place;
        /* u = 0 and a unit of nothing but what counts as nothing one by one */
        return find(p.vocab, [&](int i) { return load_any(row, DT, i); },
                    [&](int i, float x) { return counted(weight(i, x)); }, 0.0, -1.0, u).place;
    }

    /* A token drawn from max(p - q, 0), as from_row.  The rows' sums in 64 bits are known when all
     * their logits have been seen; in which tokens p is larger is known before, but for those where
     * the two are as near to each other as fp32 sums may be wrong (one or two of 151936).  So a
     * unit's part is kept as the sums of p's and of q's exponentials over the tokens where p is
     * surely larger, and over those in between with the least and the largest of their quotients, to
     * be scaled and subtracted when the sums are known.  The last workgroup weighs a unit again whose
     * quotients lie to both sides of the border then.  (Two launches instead, of both rows' sums and
     * then of their differences, took 24 and 21 us for 64 sequences, this 29.)  Exponentials are
     * summed by a product with 0 or 1: one select a token instead of four. */
    static __device__ __forceinline__ int from_rest(const AcceptParams& p, const Sequence& s,
                                                    const Draw& d, int b, int chunk, double u) {
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        const char* row = target_row(p, b, d.row);
        const char* other = draft_row(p, b, d.row);
        const Powers e(s.t, d.p_top), f(s.dt, d.q_top);
        const double ratio = uniform(d.q_sum / d.p_sum);
        uint64_t* sums = p.sums + (int64_t)b * p.sums_apart;
        uint64_t* totals = p.totals + 2 * (int64_t)b * p.chunks.by;
        const auto is_more = [&](double a, double c) { return fma(a, ratio, -c) > c * p.near; };
        const auto is_close = [&](double a, double c) {
            return fabs(fma(a, ratio, -c)) <= c * p.near && a > kNothing;
        };
        double p_sum = 0.0, q_sum = 0.0;
        for (int unit = chunk * kWaves + wave; unit < p.units; unit += p.chunks.by * kWaves) {
            const int i = unit * kUnit + lane * kN;
            const u32x4_t v = load(row, i, p.vocab), w = load(other, i, p.vocab);
            float x[kN], y[kN];
            widen(v, x);
            widen(w, y);
            double p_more = 0.0, q_more = 0.0;
            bool close = false;
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const double a = e(x[j]), c = f(y[j]);
                const double more = is_more(a, c) ? 1.0 : 0.0;
                close |= is_close(a, c);
                p_sum += a;
                q_sum += c;
                p_more = fma(a, more, p_more);
                q_more = fma(c, more, q_more);
            }
            double part = wave_sums(p_more, q_more);
            /* of the tokens in between: their sums, and the least and largest a / c */
            double between = 0.0, least = __builtin_inf(), most = 0.0;
            if (__ballot(close)) {
                double p_between = 0.0, q_between = 0.0;
#pragma unroll 1
                for (int j = 0; j < kN; ++j) {
                    const int at = min(i + j, p.vocab - 1);
                    const double a = e(load_any(row, DT, at)), c = f(load_any(other, DT, at));
                    if (i + j >= p.vocab || !is_close(a, c)) continue;
                    p_between += a;
                    q_between += c;
                    least = fmin(least, a / c);
                    most = fmax(most, a / c);
                }
                between = wave_sums(p_between, q_between);
                for (int d = 1; d < 64; d *= 2) {
                    least = fmin(least, __shfl_xor(least, d));
                    most = fmax(most, __shfl_xor(most, d));
                }
            }
            /* a unit's six numbers at once: p's and q's lie in the lanes' halves */
            const int half = lane / 32, k = lane % 32;
            if (k == 1) part = between;
            if (k == 2) part = half ? most : least;
            if (k < 3) put(&sums[6 * (int64_t)unit + 2 * k + half], part);
        }
        block_sums(p_sum, q_sum);
        if (threadIdx.x == 0) {
            put(&totals[2 * chunk], p_sum);
            put(&totals[2 * chunk + 1], q_sum);
        }
        if (!last(p, b)) return -1;
        p_sum = q_sum = 0.0;
        for (int i = threadIdx.x; i < p.chunks.by; i += DFQ_KV_THREADS) {
            p_sum += got(&totals[2 * i]);
            q_sum += got(&totals[2 * i + 1]);
        }
        double by = 0.0, draft_by = 0.0, border = 0.0;
        bool known = false;
        const auto scale = [&] {
            if (known) return;
            known = true;
            block_sums(p_sum, q_sum);
            by = 1.0 / p_sum;
            draft_by = 1.0 / q_sum;
            border = p_sum / q_sum;
        };
        const auto rest = [&](double a, double c) {
            /* both rounded: a product fused with the difference leaves its rounding where p = q */
#pragma clang fp contract(off)
            return fmax(a * by - c * draft_by, 0.0);
        };
        struct Part {
            double p, q, p_between, q_between, least, most;
        };
        const Search unit = find(p.units, [&](int i) {
            const uint64_t* v = &sums[6 * (int64_t)i];
            return Part{got(v), got(v + 1), got(v + 2), got(v + 3), got(v + 4), got(v + 5)};
        }, [&](int i, const Part& part) {
            scale();   /* here: units' parts are on their way meanwhile */
            /* p is larger where a / c is above p's sum over q's */
            double weight = rest(part.p, part.q);
            const bool above = part.least > border * (1.0 + 0x1p-48);
            if (above && part.most > 0.0) weight += rest(part.p_between, part.q_between);
            uint64_t close = __ballot(!above && part.most > border * (1.0 - 0x1p-48));
            while (close) {
                const int at = __shfl(i, __builtin_ctzll(close)), first = at * kUnit + lane * kN;
                float x[kN], y[kN];
                widen(load(row, first, p.vocab), x);
                widen(load(other, first, p.vocab), y);
                double sum = 0.0;
#pragma unroll
                for (int j = 0; j < kN; ++j) sum += rest(e(x[j]), f(y[j]));
                sum = wave_sum(sum);
                if (i == at) weight = sum;
                close &= ~__ballot(i == at);
            }
            return weight;
        }, 0.0, -1.0, u);
        if (unit.place != kNone) {
            struct Two {
                float x, y;
            };
            int from = unit.place * kUnit;
            const auto both = [&](int i) {
                return Two{load_any(row, DT, from + i), load_any(other, DT, from + i)};
            };
            int place = find(min(kUnit, p.vocab - from), both, [&](int, const Two& v) {
                return rest(e(v.x), f(v.y));
            }, unit.front, unit.goal, u).place;
            if (place == kNone) {
                from = 0;   /* as in from_row */
                place = find(p.vocab, both, [&](int, const Two& v) {
                    return counted(rest(e(v.x), f(v.y)));
                }, 0.0, -1.0, u).place;
            }
            if (place != kNone) return from + place;
        }
        /* p = q to the last bit, and yet refused (no token of the vocabulary, or a random number
         * that is not below 1): p */
        return find(p.vocab, [&](int i) { return load_any(row, DT, i); },
                    [&](int, float x) { return counted(e(x)); }, 0.0, -1.0, u).place;
    }

    static __device__ __forceinline__ void weigh(const AcceptParams& p) {
        const int b = divided(blockIdx.x, p.chunks), chunk = blockIdx.x - b * p.chunks.by;
        const Sequence s = sequence_of(p, b);
        const double u = p.uniforms[(int64_t)b * p.rows + p.rows - 1];
        const Draw d = decide(p, s, b, chunk == 0);
        int32_t* out = p.tokens + (int64_t)b * p.rows + d.row;
        if (d.mode == kDrawNone) {
            if (chunk == 0 && threadIdx.x == 0) *out = d.token;
            return;
        }
        int token;
        if (d.mode == kDrawRest) {
            token = from_rest(p, s, d, b, chunk, u);
        } else {
            const int without = d.mode == kDrawOther ? d.draft : -1;
            token = from_row(p, target_row(p, b, d.row), Powers(s.t, d.p_top), without, b, chunk, u);
            if (token == kNone) token = d.draft;   /* which has all of p */
        }
        if (token >= 0 && threadIdx.x == 0) *out = token;
    }
};

}  // namespace

#define DFQ_ACCEPT_KERNEL(op, name, call)                                          \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void                   \
        dfq_accept_##op##_##name(AcceptParams p) {                                 \
        call(p);                                                                   \
    }
#define DFQ_ACCEPT_KERNELS(name, dt)                                               \
    DFQ_ACCEPT_KERNEL(sums, name, (Accept<dt>::sums))                              \
    DFQ_ACCEPT_KERNEL(weigh, name, (Accept<dt>::weigh))
DFQ_ACCEPT_KERNELS(bf16, 0)
DFQ_ACCEPT_KERNELS(f16, 1)
DFQ_ACCEPT_KERNELS(f32, 2)
