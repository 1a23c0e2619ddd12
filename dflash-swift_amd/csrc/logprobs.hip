/*
 * logprobs.hip -- gfx950 kernels of the log probabilities of given tokens, with the entropy and
 * the top alternatives of each row of logits.
 *
 * With m the largest logit of a row and l = sum e^(x - m): the log probability of token t is
 * x_t - m - log l, the entropy log l - sum (x - m) e^(x - m) / l, in fp32.  A token of
 * probability 0 (a logit of -inf) adds nothing to the entropy.  Alternatives are ordered by
 * logit, ties to the lowest index, NaN left out.
 *
 * One pass: a wave takes a range of a row, each lane with its own running maximum and sums, and
 * keeps the range's best logits in LDS.  A workgroup's first wave joins its four; where a row has
 * several workgroups a second kernel joins theirs.
 *
 * Bound by the read of the logits where there are many: 2048 rows of 151936 in bf16 (622 MB) take
 * 120 us with up to 5 alternatives (5.2 TB/s, a large copy's rate), 129 with 20 and 137 with 32,
 * whose candidates are issue-bound work between the loads.  Few rows: two launches, 8 rows with 5
 * alternatives 7.3 and 4.3 us.
 */
#include "logit_piece.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWaves = DFQ_KV_THREADS / 64;
constexpr int kKept = 64;            /* candidates that stay without being sorted      */
constexpr int kPiece = 8;            /* most logits (or keys) that a lane brings at once */
constexpr int kRoom = kKept + 64 * kPiece;

/* Order of a logit: larger first, then the lower index; NaN below every number (0). */
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) {
    return x != x ? 0 : (uint64_t)order_of(x) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ uint64_t lanes_below(uint64_t mask, int lane) {
    return __popcll(mask & ((1ull << lane) - 1));
}

/* The best `top` keys of what a wave has met, in LDS.  All members are the same in every lane. */
struct Best {
    uint64_t* keys;      /* kRoom of them; the first `count` hold keys, in no order         */
    int count, top;
    uint64_t least;      /* keys up to it are out: the top-th best met so far, or 0         */
    float floor;         /* logits below it are out                                         */

    __device__ __forceinline__ void start(uint64_t* room, int k) {
        keys = room;
        count = 0;
        top = k;
        least = 0;
        floor = -__builtin_inff();
    }

    __device__ __forceinline__ void push(uint64_t key, int lane) {
        const bool in = key > least;
        const uint64_t mask = __ballot(in);
        if (in) keys[count + lanes_below(mask, lane)] = key;
        count += __popcll(mask);
    }

    /* A number that at least `top` of the lanes' order values reach (0 if fewer are not 0): the
     * largest with zero low bits, found bit by bit. */
    template <int LOW, int N>
    __device__ __forceinline__ uint32_t reach(const uint32_t (&order)[N]) const {
        uint32_t t = 0;
#pragma unroll
        for (int bit = 31; bit >= LOW; --bit) {
            const uint32_t c = t | 1u << bit;
            int n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) n += __popcll(__ballot(order[i] >= c));
            if (n >= top) t = c;
        }
        return t;
    }

    __device__ __forceinline__ void raise_floor(uint32_t order) {
        if (order > 0x007fffffu) floor = fmaxf(floor, key_value((uint64_t)order << 32));
    }

    /* Sorts what is held, the best first, and drops all past `top`.  Lanes hold their keys in
     * registers; those under the top-th best lane maximum go, and what is left, mostly no more
     * than a lane each, is ranked by counting. */
    template <int LOW>
    __device__ __forceinline__ void sort(int lane) {
        constexpr int kEach = kRoom / 64;
        wave_fence();
        uint64_t mine[kEach], best = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = lane + 64 * j;
            mine[j] = i < count ? keys[i] : 0;
            best = mine[j] > best ? mine[j] : best;
        }
        if (count > 64) {
            const uint32_t order[1] = {(uint32_t)(best >> 32)};
            const uint64_t t = (uint64_t)reach<LOW>(order) << 32;
            wave_fence();
            count = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const bool in = mine[j] >= t && mine[j];
                const uint64_t mask = __ballot(in);
                if (in) keys[count + lanes_below(mask, lane)] = mine[j];
                count += __popcll(mask);
            }
            wave_fence();
        }
        if (count <= 64) {
            const uint64_t key = lane < count ? keys[lane] : 0;
            int rank = 0;
            for (int i = 0; i < count; ++i) rank += keys[i] > key;
            wave_fence();
            if (lane < count && rank < top) keys[rank] = key;
        } else {
            /* many equal or rising logits: the best of all lanes, `top` times */
            uint64_t last = ~0ull, out = 0;
            for (int k = 0; k < top; ++k) {
                best = 0;
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    if (mine[j] < last && mine[j] > best) best = mine[j];
                for (int d = 1; d < 64; d *= 2) {
                    const uint64_t o = __shfl_xor((unsigned long long)best, d);
                    best = o > best ? o : best;
                }
                last = best;
                if (lane == k) out = best;
            }
            wave_fence();
            if (lane < top) keys[lane] = out;
        }
        wave_fence();
        if (count >= top) {
            count = top;
            const uint64_t k = keys[top - 1];
            /* the same in every lane, and known to be */
            const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(k >> 32));
            const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)k);
            least = (uint64_t)hi << 32 | lo;
            floor = fmaxf(floor, key_value(least));
        }
    }
};

/* Running maximum, sum of e^(x - m) and sum of (x - m) e^(x - m). */
struct Sums {
    float m, l, e;
    __device__ __forceinline__ void start() {
        m = -__FLT_MAX__;   /* not -inf: differences with it stay numbers */
        l = e = 0.0f;
    }
    __device__ __forceinline__ void raise(float to) {
        /* clamped as the logits are: past 2^-1000 the factor is 0 */
        const float d = fmaxf(m - to, -1000.0f), f = __builtin_amdgcn_exp2f(d * kLog2e);
        e = f * fmaf(d, l, e);
        l *= f;
        m = to;
    }
    __device__ __forceinline__ void add(float x) {
        const float d = x - m, w = __builtin_amdgcn_exp2f(d * kLog2e);
        l += w;
        e = fmaf(fmaxf(d, -1000.0f), w, e);   /* -inf adds 0, NaN reaches l */
    }
    __device__ __forceinline__ void join(float om, float ol, float oe) {
        const float to = fmaxf(m, om);
        Sums o = {om, ol, oe};
        raise(to);
        o.raise(to);
        l += o.l;
        e += o.e;
    }
};

template <int DT>
struct Pieces : LogitPiece<DT> {
    using LogitPiece<DT>::kN, LogitPiece<DT>::load, LogitPiece<DT>::widen,
        LogitPiece<DT>::largest;
    static constexpr int kLow = DT == 2 ? 4 : 16;    /* bits that reach() leaves        */
    static constexpr int kAhead = 4;                 /* loads in flight a lane          */

    /* The logits of 64 lanes' pieces into the sums and, where any may be among the best, into
     * them. */
    static __device__ __forceinline__ void take(u32x4_t v, int i, int end, int lane, Sums& s,
                                                Best& b) {
        float x[kN];
        widen(v, x);
        const float m = largest(x);
        if (m > s.m) s.raise(m);
#pragma unroll
        for (int j = 0; j < kN; ++j) s.add(x[j]);
        if (b.top == 0) return;
        if (!__any(m >= b.floor)) return;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const bool in = i + j < end && x[j] >= b.floor;
            if (__any(in)) b.push(in ? order_key(x[j], (uint32_t)(i + j)) : 0, lane);
        }
        if (b.count > kKept) b.sort<kLow>(lane);
    }

    static __device__ __forceinline__ void part(const LogprobParams& p) {
        __shared__ uint64_t room[kWaves][kRoom];
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        const int r = blockIdx.x / p.splits, parts = p.splits * kWaves;
        const int part = blockIdx.x % p.splits * kWaves + wave;
        const char* row = (const char*)p.logits + (int64_t)r * p.row_stride * (16 / kN);
        constexpr int kStep = 64 * kN;
        const int steps = (p.vocab + kStep - 1) / kStep;
        const int each = (steps + parts - 1) / parts;
        const int from = part * each * kStep < p.vocab ? part * each * kStep : p.vocab;
        const int end = each * kStep < p.vocab - from ? from + each * kStep : p.vocab;
        Sums s;
        s.start();
        Best b;
        b.start(room[wave], p.top);
        /* Each lane's largest logit so far, as its order value (0: none).  What `top` lanes of
         * the workgroup have reached is a floor for all of its waves, whenever it is looked at.
         * It is set by the first logits and raised each time their number has doubled: without
         * the other waves' lanes and the later looks, 2048 rows of 151936 with 20 alternatives
         * took 156 us for 129, 32 alternatives 183 for 137. */
        __shared__ uint32_t reached[kWaves][64];
        int turn = 0, due = 0;
        for (int at = from; turn == 0 || at < end; at += kAhead * kStep, ++turn) {
            u32x4_t v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                v[u] = load(row, at + u * kStep + lane * kN, end);
            if (p.top && turn == due) {
                if (turn == 0) {
                    float m = -__builtin_inff();
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        float x[kN];
                        widen(v[u], x);
                        m = fmaxf(m, largest(x));
                    }
                    if (m > s.m) s.raise(m);
                }
                __hip_atomic_store(&reached[wave][lane], s.m > -__FLT_MAX__ ? order_of(s.m) : 0,
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (turn == 0) __syncthreads();
                uint32_t order[kWaves];
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
                    order[w] = __hip_atomic_load(&reached[w][lane], __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_WORKGROUP);
                b.raise_floor(b.reach<kLow>(order));
                due = 2 * turn + 1;
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (at + u * kStep >= end) break;
                take(v[u], at + u * kStep + lane * kN, end, lane, s, b);
            }
        }
        for (int d = 1; d < 64; d *= 2)
            s.join(__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.e, d));
        /* the waves' sums and candidates together, by the first wave */
        __shared__ f32x4_t sums[kWaves];
        __shared__ int counts[kWaves];
        if (lane == 0) {
            sums[wave] = f32x4_t{s.m, s.l, s.e, 0.0f};
            counts[wave] = b.count;
        }
        __syncthreads();
        if (wave != 0) return;
        for (int w = 1; w < kWaves; ++w) {
            s.join(sums[w][0], sums[w][1], sums[w][2]);
            if (p.top == 0) continue;
            const int n = __builtin_amdgcn_readfirstlane(counts[w]);   /* at most kKept */
            b.push(lane < n ? room[w][lane] : 0, lane);
            if (b.count > kKept) b.sort<kLow>(lane);
        }
        if (p.top) b.sort<kLow>(lane);
        if (p.splits == 1) return finish(p, r, lane, s, b);
        if (lane == 0)
            *(f32x4_t*)(p.part_sums + (int64_t)blockIdx.x * 4) = f32x4_t{s.m, s.l, s.e, 0.0f};
        if (lane < p.top)
            p.part_keys[(int64_t)blockIdx.x * p.top + lane] = lane < b.count ? b.keys[lane] : 0;
    }

    /* A row's parts together, by one wave. */
    static __device__ __forceinline__ void join(const LogprobParams& p) {
        __shared__ uint64_t room[kRoom];
        const int lane = threadIdx.x, r = blockIdx.x;
        const f32x4_t* sums = (const f32x4_t*)p.part_sums + (int64_t)r * p.splits;
        Sums s;
        s.start();
        for (int i = lane; i < p.splits; i += 64) {
            const f32x4_t v = sums[i];
            s.join(v[0], v[1], v[2]);
        }
        for (int d = 1; d < 64; d *= 2)
            s.join(__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.e, d));
        Best b;
        b.start(room, p.top);
        const int n = p.splits * p.top;
        const uint64_t* keys = p.part_keys + (int64_t)r * n;
        if (n > 64 * kPiece) {
            /* What `top` lanes reach is a floor here too, and few keys are left to sort: 16 rows
             * with 32 alternatives 30.4 -> 23.1 us.  Keys of one piece are sorted sooner than it
             * is found (33 rows with one 10.2 us, with it 10.8). */
            uint32_t most[1] = {0};
            for (int i = lane; i < n; i += 64) {
                const uint32_t order = (uint32_t)(keys[i] >> 32);
                most[0] = order > most[0] ? order : most[0];
            }
            const uint32_t reached = b.reach<kLow>(most);
            if (reached) b.least = ((uint64_t)reached << 32) - 1;
        }
        for (int at = 0; at < n; at += 64 * kPiece) {
            uint64_t k[kPiece];
#pragma unroll
            for (int j = 0; j < kPiece; ++j) {
                const int i = at + j * 64 + lane;
                k[j] = i < n ? keys[i] : 0;
            }
#pragma unroll
            for (int j = 0; j < kPiece; ++j)
                if (at + j * 64 < n) b.push(k[j], lane);
            if (b.count > kKept) b.sort<kLow>(lane);
        }
        if (p.top) b.sort<kLow>(lane);
        finish(p, r, lane, s, b);
    }

    /* A row's outputs from its sums and its best, sorted. */
    static __device__ __forceinline__ void finish(const LogprobParams& p, int r, int lane,
                                                  const Sums& s, const Best& b) {
        /* no number above -inf: no distribution */
        const float log_l = s.l > 0.0f ? logf(s.l) : __builtin_nanf("");
        if (lane == 0) {
            if (p.entropy) p.entropy[r] = log_l - s.e / s.l;
            if (p.tokens) {
                const int t = p.tokens[r];
                const char* row = (const char*)p.logits + (int64_t)r * p.row_stride * (16 / kN);
                p.logprobs[r] = t >= 0 && t < p.vocab ? load_any(row, DT, t) - s.m - log_l
                                                      : __builtin_nanf("");
            }
        }
        if (lane < p.top) {
            const bool has = lane < b.count;
            const uint64_t k = b.keys[lane];
            p.top_tokens[(int64_t)r * p.top + lane] = has ? (int32_t)~(uint32_t)k : -1;
            p.top_logprobs[(int64_t)r * p.top + lane] =
                has ? key_value(k) - s.m - log_l : __builtin_nanf("");
        }
    }
};

}  // namespace

#define DFQ_LOGPROB_KERNELS(name, dt)                                            \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void                 \
        dfq_token_logprobs_##name(LogprobParams p) {                             \
        Pieces<dt>::part(p);                                                     \
    }                                                                            \
    extern "C" __global__ __launch_bounds__(64) void                             \
        dfq_token_logprobs_join_##name(LogprobParams p) {                        \
        Pieces<dt>::join(p);                                                     \
    }
DFQ_LOGPROB_KERNELS(bf16, 0)
DFQ_LOGPROB_KERNELS(f16, 1)
DFQ_LOGPROB_KERNELS(f32, 2)
