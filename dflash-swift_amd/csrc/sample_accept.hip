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
 * The draw is a whole number that a sum's last bits decide, so all that it comes from is 64 bits
 * wide: sums of 2^x over the row, and the running sum.  The accept's sums over all rows are fp32:
 * a draft's chance is then right to some 2^-21 of itself.
 */
#include "kv_params.h"
#include "logit_piece.h"

namespace {

constexpr int kWaves = DFQ_KV_THREADS / 64;
constexpr double kLog2e = 1.44269504088896340736;

/* 2^a for a <= 0: the Taylor sum of the part behind the whole number, whose first term left out
 * is (ln 2 / 2)^12 / 12! < 7e-15. */
__device__ __forceinline__ double power_of_2(double a) {
    a = fmax(a, -1100.0);
    const double n = rint(a), x = (a - n) * 0.693147180559945309417;
    double s = 1.0 / 39916800.0;
    s = fma(x, s, 1.0 / 3628800.0);
    s = fma(x, s, 1.0 / 362880.0);
    s = fma(x, s, 1.0 / 40320.0);
    s = fma(x, s, 1.0 / 5040.0);
    s = fma(x, s, 1.0 / 720.0);
    s = fma(x, s, 1.0 / 120.0);
    s = fma(x, s, 1.0 / 24.0);
    s = fma(x, s, 1.0 / 6.0);
    s = fma(x, s, 0.5);
    s = fma(x, s, 1.0);
    s = fma(x, s, 1.0);
    return __builtin_ldexp(s, (int)n);
}

/* Temperatures below the least normal number are taken for it: their reciprocal is finite, and
 * the logits' differences pass any exponent with either. */
__device__ __forceinline__ double rate_of(float t) {
    return kLog2e / (double)fmaxf(t, 1.17549435e-38f);
}
__device__ __forceinline__ bool is_temperature(float t) {
    return t >= 0.0f && t < __builtin_inff();
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

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double waves[kWaves];
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += waves[w];
    __syncthreads();
    return s;
}

/* The largest logit with its place, and the sum of e^((x - max(top, -FLT_MAX)) / T). */
struct RowSums {
    float m, l, top;
    int at;
    __device__ __forceinline__ void start() {
        m = -__FLT_MAX__;   /* not -inf: differences with it stay numbers */
        l = 0.0f;
        top = -__builtin_inff();
        at = -1;
    }
    __device__ __forceinline__ void join(const RowSums& o, float rate) {
        const float to = fmaxf(m, o.m);
        l = l * __builtin_amdgcn_exp2f((m - to) * rate) +
            o.l * __builtin_amdgcn_exp2f((o.m - to) * rate);
        m = to;
        if (o.at >= 0 && (at < 0 || o.top > top || (o.top == top && o.at < at))) {
            top = o.top;
            at = o.at;
        }
    }
};

template <int DT>
struct Accept : LogitPiece<DT> {
    using LogitPiece<DT>::kN, LogitPiece<DT>::load, LogitPiece<DT>::widen,
        LogitPiece<DT>::largest;
    static constexpr int kSize = 16 / kN, kAhead = 4;
    static constexpr int kChunk = DFQ_KV_THREADS * kN;

    static __device__ __forceinline__ const char* target_row(const AcceptParams& p, int b, int r) {
        return (const char*)p.logits + (b * p.batch_stride + r * p.row_stride) * kSize;
    }
    static __device__ __forceinline__ const char* draft_row(const AcceptParams& p, int b, int r) {
        return (const char*)p.draft_logits +
               (b * p.draft_batch_stride + r * p.draft_row_stride) * kSize;
    }

    /* One range of one row. */
    static __device__ __forceinline__ void sums(const AcceptParams& p) {
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        const int split = blockIdx.x % p.splits, row = blockIdx.x / p.splits;
        const int b = row / p.all_rows, r = row % p.all_rows;
        const bool draft = r >= p.rows;
        const Sequence q = sequence_of(p, b);
        /* rows behind a sequence's drafts, and draft rows that do not matter */
        if (draft ? r - p.rows >= q.drafts || !q.drafted : r > q.drafts) return;
        const char* at_row = draft ? draft_row(p, b, r - p.rows) : target_row(p, b, r);
        const float t = draft ? q.dt : q.t;
        const float rate = t > 0.0f ? (float)rate_of(t) : 0.0f;
        constexpr int kStep = 64 * kN;
        const int steps = (p.vocab + kStep - 1) / kStep, parts = p.splits * kWaves;
        const int each = (steps + parts - 1) / parts, part = split * kWaves + wave;
        const int from = (int64_t)part * each * kStep < p.vocab ? part * each * kStep : p.vocab;
        const int end = each * kStep < p.vocab - from ? from + each * kStep : p.vocab;
        RowSums s;
        s.start();
        for (int at = from; at < end; at += kAhead * kStep) {
            u32x4_t v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) v[u] = load(at_row, at + u * kStep + lane * kN, end);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = at + u * kStep + lane * kN;
                float x[kN];
                widen(v[u], x);
                const float m = largest(x);
                if (m > s.top || (s.at < 0 && m == s.top && i < end)) {
                    s.top = m;
#pragma unroll
                    for (int j = kN - 1; j >= 0; --j)
                        if (x[j] == m && i + j < end) s.at = i + j;
                    if (m > s.m) {
                        s.l *= __builtin_amdgcn_exp2f((s.m - m) * rate);
                        s.m = m;
                    }
                }
#pragma unroll
                for (int j = 0; j < kN; ++j)
                    s.l += __builtin_amdgcn_exp2f((x[j] - s.m) * rate);
            }
        }
        for (int d = 1; d < 64; d *= 2) {
            const RowSums o = {__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.top, d),
                               __shfl_xor(s.at, d)};
            s.join(o, rate);
        }
        __shared__ RowSums waves[kWaves];
        if (lane == 0) waves[wave] = s;
        __syncthreads();
        if (threadIdx.x) return;
        for (int w = 1; w < kWaves; ++w) s.join(waves[w], rate);
        p.parts[blockIdx.x] = AcceptPart{s.top, s.l, s.at, 0};
    }

    /* A row's parts together; sum is NaN or 0 where the row has no distribution. */
    struct Row {
        float top;
        double sum;
        int at;
    };
    static __device__ __forceinline__ Row row_of(const AcceptParams& p, int b, int r, float t) {
        const AcceptPart* part = p.parts + ((int64_t)b * p.all_rows + r) * p.splits;
        Row row = {-__builtin_inff(), 0.0, -1};
        for (int i = 0; i < p.splits; ++i)
            if (part[i].at >= 0 && (row.at < 0 || part[i].top > row.top)) {
                row.top = part[i].top;
                row.at = part[i].at;
            }
        const double rate = t > 0.0f ? rate_of(t) : 0.0;
        const float top = fmaxf(row.top, -__FLT_MAX__);
        for (int i = 0; i < p.splits; ++i)
            row.sum += part[i].sum *
                       power_of_2(((double)fmaxf(part[i].top, -__FLT_MAX__) - top) * rate);
        return row;
    }

    /* What a wave decides of a sequence: lane i looks at draft i. */
    static __device__ __forceinline__ void decide(const AcceptParams& p) {
        const int b = blockIdx.x, lane = threadIdx.x;
        const Sequence s = sequence_of(p, b);
        const bool greedy = s.t == 0.0f;
        Row row = {0.0f, 0.0, -1}, other = row;
        float chance = 0.0f;
        bool some = true, taken = false;   /* some: both rows have a distribution */
        int draft = -1;
        if (lane <= s.drafts) {
            row = row_of(p, b, lane, s.t);
            some = greedy ? row.at >= 0 : row.sum > 0.0 && row.sum < __builtin_inf() &&
                                              is_temperature(s.t);
            if (lane < s.drafts) {
                draft = p.drafts[(int64_t)b * (p.rows - 1) + lane];
                const bool known = draft >= 0 && draft < p.vocab;
                double mine = 0.0, theirs = 1.0;
                if (s.drafted) {
                    other = row_of(p, b, p.rows + lane, s.dt);
                    some = some && other.sum > 0.0 && other.sum < __builtin_inf() &&
                           is_temperature(s.dt);
                }
                if (known && some) {
                    if (greedy)
                        mine = draft == row.at;
                    else
                        mine = power_of_2(((double)load_any(target_row(p, b, lane), DT, draft) -
                                           row.top) * rate_of(s.t)) / row.sum;
                    if (s.drafted)
                        theirs = power_of_2(((double)load_any(draft_row(p, b, lane), DT, draft) -
                                             other.top) * rate_of(s.dt)) / other.sum;
                    taken = (double)p.uniforms[(int64_t)b * p.rows + lane] * theirs < mine;
                    chance = theirs > 0.0 ? (float)fmin(mine / theirs, 1.0) : mine > 0.0;
                }
            }
        }
        if (p.chances && lane < p.rows - 1)
            p.chances[(int64_t)b * (p.rows - 1) + lane] = chance;
        const uint64_t refused = ~__ballot(taken);
        const int n = __builtin_ctzll(refused);   /* at most 63 drafts: some bit is set */
        int token = lane < n ? draft : -1;
        if (lane == n) {
            AcceptDraw d = {DFQ_DRAW_NONE, n, draft, row.top, other.top, 0};
            if (!some) {
                token = -1;
            } else if (greedy) {
                token = row.at;
            } else if (n == s.drafts) {
                d.mode = DFQ_DRAW_P;
            } else {
                d.mode = s.drafted ? DFQ_DRAW_REST : DFQ_DRAW_OTHER;
            }
            p.draws[b] = d;
            p.accepted[b] = n;
        }
        if (lane < p.rows) p.tokens[(int64_t)b * p.rows + lane] = token;
    }

    /* Terms of the sums over a chunk's lane: e^((x - top) / T) in 64 bits. */
    static __device__ __forceinline__ void terms(const char* row, int i, int end, float top,
                                                 double rate, double (&w)[kN]) {
        float x[kN];
        widen(load(row, i, end), x);
#pragma unroll
        for (int j = 0; j < kN; ++j) w[j] = power_of_2(((double)x[j] - top) * rate);
    }

    /* Both rows' sums over a chunk, where the draw is from their difference. */
    static __device__ __forceinline__ void totals(const AcceptParams& p) {
        const int b = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
        const AcceptDraw d = p.draws[b];
        if (d.mode != DFQ_DRAW_REST) return;
        const Sequence s = sequence_of(p, b);
        const int i = chunk * kChunk + (int)threadIdx.x * kN;
        for (int k = 0; k < 2; ++k) {
            double w[kN], sum = 0.0;
            terms(k ? draft_row(p, b, d.row) : target_row(p, b, d.row), i, p.vocab,
                  k ? d.q_top : d.p_top, rate_of(k ? s.dt : s.t), w);
#pragma unroll
            for (int j = 0; j < kN; ++j) sum += w[j];
            sum = block_sum(sum);
            if (threadIdx.x == 0) p.totals[((int64_t)b * 2 + k) * p.chunks + chunk] = sum;
        }
    }

    /* The sum of a sequence's chunks. */
    static __device__ __forceinline__ double sum_of(const double* sums, int chunks) {
        double v = 0.0;
        for (int i = threadIdx.x; i < chunks; i += DFQ_KV_THREADS) v += sums[i];
        return block_sum(v);
    }

    /* What a lane's logits of a chunk weigh in the draw; p_by and q_by are 1 / sums (REST). */
    static __device__ __forceinline__ void weigh(const AcceptParams& p, const AcceptDraw& d,
                                                 const Sequence& s, int b, int chunk, double p_by,
                                                 double q_by, double (&w)[kN]) {
        const int i = chunk * kChunk + (int)threadIdx.x * kN;
        terms(target_row(p, b, d.row), i, p.vocab, d.p_top, rate_of(s.t), w);
        if (d.mode == DFQ_DRAW_OTHER) {
#pragma unroll
            for (int j = 0; j < kN; ++j)
                if (i + j == d.draft) w[j] = 0.0;
        }
        if (d.mode == DFQ_DRAW_REST) {
            double q[kN];
            terms(draft_row(p, b, d.row), i, p.vocab, d.q_top, rate_of(s.dt), q);
#pragma unroll
            for (int j = 0; j < kN; ++j) w[j] = fmax(w[j] * p_by - q[j] * q_by, 0.0);
        }
    }

    static __device__ __forceinline__ void weights(const AcceptParams& p) {
        const int b = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
        const AcceptDraw d = p.draws[b];
        if (d.mode == DFQ_DRAW_NONE) return;
        const Sequence s = sequence_of(p, b);
        double p_by = 0.0, q_by = 0.0;
        if (d.mode == DFQ_DRAW_REST) {
            const double* t = p.totals + (int64_t)b * 2 * p.chunks;
            p_by = 1.0 / sum_of(t, p.chunks);
            q_by = 1.0 / sum_of(t + p.chunks, p.chunks);
        }
        double w[kN], sum = 0.0;
        weigh(p, d, s, b, chunk, p_by, q_by, w);
#pragma unroll
        for (int j = 0; j < kN; ++j) sum += w[j];
        sum = block_sum(sum);
        if (threadIdx.x == 0) p.weights[(int64_t)b * p.chunks + chunk] = sum;
    }

    /* The token of a sequence, by one workgroup: its chunk, then its place in it. */
    static __device__ __forceinline__ void pick(const AcceptParams& p) {
        const int b = blockIdx.x;
        AcceptDraw d = p.draws[b];
        if (d.mode == DFQ_DRAW_NONE) return;
        const Sequence s = sequence_of(p, b);
        const double* sums = p.weights + (int64_t)b * p.chunks;
        const double* t = p.totals + (int64_t)b * 2 * p.chunks;
        int32_t* out = p.tokens + (int64_t)b * p.rows + d.row;
        double all = sum_of(sums, p.chunks), p_by = 0.0, q_by = 0.0;
        if (d.mode == DFQ_DRAW_REST) {
            if (all > 0.0) {
                p_by = 1.0 / sum_of(t, p.chunks);
                q_by = 1.0 / sum_of(t + p.chunks, p.chunks);
            } else {   /* p = q: nothing is left of p */
                d.mode = DFQ_DRAW_P;
                sums = t;
                all = sum_of(sums, p.chunks);
            }
        }
        if (d.mode == DFQ_DRAW_OTHER && !(all > 0.0)) {   /* the draft has all of p */
            if (threadIdx.x == 0) *out = d.draft;
            return;
        }
        const double goal = (double)p.uniforms[(int64_t)b * p.rows + p.rows - 1] * all;
        __shared__ int chunk, place[2];
        __shared__ double before;
        if (threadIdx.x == 0) {
            /* the first whose running sum passes the goal, or the last that weighs anything */
            double sum = 0.0;
            chunk = 0;
            before = 0.0;
            for (int i = 0; i < p.chunks; ++i) {
                if (sums[i] > 0.0) {
                    chunk = i;
                    before = sum;
                }
                sum += sums[i];
                if (sum > goal) break;
            }
            place[0] = 0x7fffffff;
            place[1] = 0;
        }
        __syncthreads();
        double w[kN], sum = 0.0;
        weigh(p, d, s, b, chunk, p_by, q_by, w);
#pragma unroll
        for (int j = 0; j < kN; ++j) sum += w[j];
        /* the lanes' sums in order */
        __shared__ double lanes[DFQ_KV_THREADS];
        lanes[threadIdx.x] = sum;
        __syncthreads();
        double run = before;
        for (int i = 0; i < (int)threadIdx.x; ++i) run += lanes[i];
        int first = 0x7fffffff, last = 0;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const int i = chunk * kChunk + (int)threadIdx.x * kN + j;
            run += w[j];
            if (w[j] > 0.0) {
                last = i;
                if (run > goal && first == 0x7fffffff) first = i;
            }
        }
        atomicMin(&place[0], first);
        atomicMax(&place[1], last);
        __syncthreads();
        if (threadIdx.x == 0) *out = place[0] != 0x7fffffff ? place[0] : place[1];
    }
};

}  // namespace

#define DFQ_ACCEPT_KERNEL(op, name, dt, threads)                                   \
    extern "C" __global__ __launch_bounds__(threads) void dfq_accept_##op##_##name( \
        AcceptParams p) {                                                          \
        Accept<dt>::op(p);                                                         \
    }
#define DFQ_ACCEPT_KERNELS(name, dt)                    \
    DFQ_ACCEPT_KERNEL(sums, name, dt, DFQ_KV_THREADS)   \
    DFQ_ACCEPT_KERNEL(decide, name, dt, 64)             \
    DFQ_ACCEPT_KERNEL(totals, name, dt, DFQ_KV_THREADS) \
    DFQ_ACCEPT_KERNEL(weights, name, dt, DFQ_KV_THREADS) \
    DFQ_ACCEPT_KERNEL(pick, name, dt, DFQ_KV_THREADS)
DFQ_ACCEPT_KERNELS(bf16, 0)
DFQ_ACCEPT_KERNELS(f16, 1)
DFQ_ACCEPT_KERNELS(f32, 2)
