/*
 * rope.hip -- gfx950 kernels of the rotary positions of queries and keys, alone and behind the RMS
 * norm of each head.
 *
 * With f the frequencies (radians a position) of a head's R/2 rotated pairs, position p turns the
 * pair (a, b) i by the angle t = p f_i:
 *   a' = A (a cos t - b sin t),   b' = A (b cos t + a sin t),
 * channels behind R stay.  Pairs are (i, i + R/2) or, interleaved, (2i, 2i + 1).  The norm in front
 * is x (w + offset) / sqrt(mean x^2 + eps) over a head's channels.  All of it in fp32, rounded once.
 *
 * The angle of a far position has no room in fp32 (position 10^6 at a frequency of 1 is known to
 * 0.06), so frequencies are whole numbers F of 2^-64 turns: p F mod 2^64, in whole arithmetic, is
 * the angle's place in its turn, whatever p, and its upper 32 bits leave an error of 2^-32 turns.
 * Sine and cosine are their Taylor sums over an eighth of a turn to both sides of the nearest
 * quarter: the first terms left out are x^11 / 11! < 1.8e-9 and x^12 / 12! < 1.2e-10.
 *
 * Bound by memory where there are many rows, and by the launch where there are few.  A pair's angle
 * costs 30 instructions, so that a lane turns up to 16 heads of its token by the same ones, the next
 * head's channels on their way meanwhile; outputs go past the caches.  8192 rows of 40 + 8 heads of
 * 128 in bf16, cut from fused rows (201 MB): 39.5 us (5.1 TB/s, a large copy's rate), with norms
 * 40.5.  One head a lane took 57 us, up to 8 of them with plain stores 45.  One row of 8 sequences
 * 4.0 us, 8 rows with norms 4.6, 1665 rows of 18 heads of 256 with a quarter rotated 9.8 (31 MB).
 *
 * Stores past the caches have little effect on the kernels that read the outputs next.  Norms, cache
 * append and attention over 300 to 500 tokens with plain stores, then with these: 8 rows 18.4 and 18.5
 * us, 16 sequences of 8 rows 24.2 and 24.3, 64 of 8 rows 40.7 and 40.3, 64 of 16 rows 97.0 and 98.2.
 */
#include "kv_device.h"

namespace {

/* Two numbers to nearest even, the first in the low half. */
template <bool F16>
__device__ __forceinline__ uint32_t rounded2(float a, float b) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)a, (_Float16)b});
    else return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b});
}

/* Sine and cosine of t 2^-32 turns. */
__device__ __forceinline__ void turn_of(uint32_t t, float& sine, float& cosine) {
    const uint32_t quarter = (t + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(t - (quarter << 30)) * (6.28318530717958647692f * 0x1p-32f);
    const float y = x * x;
    float s = fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f);
    s = fmaf(y, s, 1.0f / 120.0f);
    s = fmaf(y, s, -1.0f / 6.0f);
    s = fmaf(x * y, s, x);
    float c = fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    c = fmaf(y, c, -1.0f / 720.0f);
    c = fmaf(y, c, 1.0f / 24.0f);
    c = fmaf(y, c, -0.5f);
    c = fmaf(y, c, 1.0f);
    sine = quarter & 1 ? c : s;
    cosine = quarter & 1 ? s : c;
    if (quarter & 2) sine = -sine;
    if ((quarter + 1) & 2) cosine = -cosine;
}

/* The position of row m of sequence b, negated where the rotation is undone. */
__device__ __forceinline__ uint64_t position(const RopeParams& p, int b, int m) {
    const int64_t pos = p.positions ? (int64_t)p.positions[(int64_t)b * p.rows.by + m]
                                    : (int64_t)p.start + (p.starts ? p.starts[b] : 0) + m;
    return (uint64_t)(p.inverse ? -pos : pos);
}

/* Sine and cosine of pair i at `pos`, times the amplitude. */
__device__ __forceinline__ void pair_turn(const RopeParams& p, uint64_t pos, int i, float& sine,
                                          float& cosine) {
    turn_of((uint32_t)(pos * p.turns[i] >> 32), sine, cosine);
    sine *= p.amplitude;
    cosine *= p.amplitude;
}

__device__ __forceinline__ void turn(float& a, float& b, float sine, float cosine) {
    const float c = a;
    a = c * cosine - b * sine;
    b = b * cosine + c * sine;
}

/* 8 neighbouring elements, as they lie in memory (heads cut from a fused projection have any offset)
 * and as fp32. */
template <int DT>
struct Chunk {
    static constexpr int kSize = DT == 2 ? 4 : 2, kWords = kSize / 2;
    u32x4_t raw[kWords];
    __device__ __forceinline__ void load(const void* base, int64_t at) {
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            raw[i] = *(const u32x4_any*)((const char*)base + at * kSize + 16 * i);
    }
    __device__ __forceinline__ void store(void* base, int64_t at) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            __builtin_nontemporal_store(raw[i],
                                        (u32x4_any*)((char*)base + at * kSize + 16 * i));
    }
    __device__ __forceinline__ void widen(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == 2) f[i] = __uint_as_float(raw[i / 4][i % 4]);
            else f[i] = elem_to_f32<DT == 1>(raw[0][i / 2] >> (16 * (i % 2)) & 0xffffu);
        }
    }
    __device__ __forceinline__ void round(const float (&f)[8]) {
        if constexpr (DT == 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i / 4][i % 4] = __float_as_uint(f[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[0][i] = rounded2<DT == 1>(f[2 * i], f[2 * i + 1]);
        }
    }
};

/* The sum over the `lanes` (a power of two) that hold a head. */
__device__ __forceinline__ float head_sum(float v, int lanes) {
    const auto add = [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    };
    uint32_t u = __float_as_uint(v);
    if (lanes > 1) u = exchange<0xB1>(u, add);
    if (lanes > 2) u = exchange<0x4E>(u, add);
    if (lanes > 4) u = exchange<0x141>(u, add);
    if (lanes > 8) u = exchange<0x140>(u, add);
    v = __uint_as_float(u);
    if (lanes > 16) v += __shfl_xor(v, 16);
    if (lanes > 32) v += __shfl_xor(v, 32);
    return v;
}

/* What a kernel norms its heads by. */
enum { kAlone, kNorm, kNormSmall };

/* The factor of a head over `lanes` lanes, 1 / sqrt(mean(x^2) + eps).
 *
 * Squares may lose bits to denormals, or all of them, where they and eps together are below
 * DFQ_NORM_SMALL on the mean: such a head's channels are lifted 2^100 fold and squared again, the least
 * number's square then a normal one (2^-98) and the largest (2^-50 sqrt(dim)) far from infinity.
 * An eps of that size rules it out for all heads, so that kernels of their own ask (kNormSmall): the
 * question took 8192 rows of 40 + 8 heads of 128 from 40.2 to 40.5 us and one block from 4.54 to
 * 4.65. */
template <int NORM, int N>
__device__ __forceinline__ float norm_factor(const RopeParams& p, float (&x)[2][N], int lanes) {
    const auto mean = [&] {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) sum = fmaf(x[0][i], x[0][i], fmaf(x[1][i], x[1][i], sum));
        return head_sum(sum, lanes) / (float)p.dim;
    };
    float square = mean() + p.eps;
    if constexpr (NORM == kNormSmall) {
        constexpr float kLift = 0x1p100f;
        if (square < DFQ_NORM_SMALL) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[0][i] *= kLift;
                x[1][i] *= kLift;
            }
            square = mean() + p.eps * kLift * kLift;
        }
    }
    return rsqrtf(square);
}

/* Heads of 16 n channels: a lane holds two chunks of 8, so that it has both channels of each of
 * its 8 pairs, of every `slots`-th head of one token, whose angles it finds once.  `lanes` lanes a
 * head, neighbouring heads side by side. */
template <int DT, int NORM, bool INTERLEAVED>
__device__ __forceinline__ void rotate_heads(const RopeParams& p) {
    const bool keys = (int)blockIdx.x >= p.q_groups;
    const RopeTensor& t = p.t[keys];
    const int group = keys ? blockIdx.x - p.q_groups : blockIdx.x;
    const int lane = threadIdx.x % p.lanes;
    const int64_t slot = (int64_t)group * (DFQ_KV_THREADS / p.lanes) + threadIdx.x / p.lanes;
    if (slot >= (int64_t)p.tokens * t.slots.by) return;
    const int token = divided((int)slot, t.slots);
    int head = (int)slot - token * t.slots.by;
    const int b = divided(token, p.rows), m = token - b * p.rows.by;
    const bool active = lane * 16 < p.dim;
    /* the lane's chunks: of a rotated half and its partner, or neighbours */
    const bool halves = !INTERLEAVED && lane * 8 < p.pairs;
    const int at0 = halves ? lane * 8 : lane * 16;
    const int at1 = halves ? at0 + p.pairs : at0 + 8;
    const int64_t in = b * t.in_batch + m * t.in_row, out = b * t.out_batch + m * t.out_row;
    Chunk<DT> c[2] = {};
    if (active) {
        c[0].load(t.in, in + head * t.in_head + at0);
        c[1].load(t.in, in + head * t.in_head + at1);
    }
    float w[2][8];
    if constexpr (NORM) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[k][i] = 1.0f;
            if (!t.weight || !active) continue;
            if (p.weight_f32) {
                Chunk<2> v;
                v.load(t.weight, k ? at1 : at0);
                v.widen(w[k]);
            } else {
                Chunk<DT> v;
                v.load(t.weight, k ? at1 : at0);
                v.widen(w[k]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) w[k][i] += p.offset;
        }
    }
    float sine[8] = {}, cosine[8] = {};
    const int pairs = active ? p.pairs - lane * 8 : 0;   /* of this lane's 8 that turn */
    if (pairs > 0) {
        const uint64_t pos = position(p, b, m);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < pairs) pair_turn(p, pos, lane * 8 + i, sine[i], cosine[i]);
    }
    for (;;) {
        float x[2][8];
        c[0].widen(x[0]);
        c[1].widen(x[1]);
        /* the next head comes meanwhile */
        const int next = head + t.slots.by;
        if (active && next < t.heads) {
            c[0].load(t.in, in + next * t.in_head + at0);
            c[1].load(t.in, in + next * t.in_head + at1);
        }
        if constexpr (NORM) {
            const float scale = norm_factor<NORM>(p, x, p.lanes);
            /* first the factor of the head, whose product with a weight fp32 need not hold */
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[0][i] = x[0][i] * scale * w[0][i];
                x[1][i] = x[1][i] * scale * w[1][i];
            }
        }
        /* channels behind the rotated ones stay as they are, infinities and NaN among them */
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= pairs) break;
            if constexpr (INTERLEAVED)
                turn(x[i / 4][2 * (i % 4)], x[i / 4][2 * (i % 4) + 1], sine[i], cosine[i]);
            else
                turn(x[0][i], x[1][i], sine[i], cosine[i]);
        }
        if (active) {
            Chunk<DT> y[2];
            y[0].round(x[0]);
            y[1].round(x[1]);
            y[0].store(t.out, out + head * t.out_head + at0);
            y[1].store(t.out, out + head * t.out_head + at1);
        }
        if (next >= t.heads) return;
        head = next;
    }
}

/* Any even head and any number of pairs: a wave a head, a lane a pair at a time.
 *
 * Bound by instructions: a wave finds its head's angles and addresses for itself, and its lanes take
 * an element at a time.  8192 rows of 40 + 8 heads of 80 with 20 or 40 channels rotated take 103 us in
 * bf16 (126 MB, 1.2 TB/s) and 109 in fp32 (twice the bytes), with norms 133 in both; heads of 96 with
 * 24 rotated 106 and 114, with norms 135 and 138. */
template <int DT, int NORM>
__device__ __forceinline__ void rotate_any(const RopeParams& p) {
    const int lane = threadIdx.x % 64;
    const bool keys = (int)blockIdx.x >= p.q_groups;
    const RopeTensor& t = p.t[keys];
    const int group = keys ? blockIdx.x - p.q_groups : blockIdx.x;
    const int64_t slot = (int64_t)group * (DFQ_KV_THREADS / 64) + threadIdx.x / 64;
    if (slot >= (int64_t)p.tokens * t.slots.by) return;
    const int token = divided((int)slot, t.slots), head = (int)slot - token * t.slots.by;
    const int b = divided(token, p.rows), m = token - b * p.rows.by;
    const int64_t from = b * t.in_batch + m * t.in_row + head * t.in_head;
    const int64_t to = b * t.out_batch + m * t.out_row + head * t.out_head;
    const uint64_t pos = position(p, b, m);
    constexpr int kMost = DFQ_ROPE_DIM / 128;   /* pairs a lane */
    float x[2][kMost];
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const int i = lane + 64 * j;
        x[0][j] = x[1][j] = 0.0f;
        if (2 * i < p.dim) {
            const bool apart = !p.interleaved && i < p.pairs;
            x[0][j] = load_any(t.in, DT, from + (apart ? i : 2 * i));
            x[1][j] = load_any(t.in, DT, from + (apart ? i + p.pairs : 2 * i + 1));
        }
    }
    float scale = 1.0f;
    if constexpr (NORM) scale = norm_factor<NORM>(p, x, 64);
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const int i = lane + 64 * j;
        if (2 * i >= p.dim) continue;
        const bool apart = !p.interleaved && i < p.pairs;
        const int at0 = apart ? i : 2 * i, at1 = apart ? i + p.pairs : 2 * i + 1;
        float a = x[0][j], c = x[1][j];
        if constexpr (NORM) {
            const int wt = p.weight_f32 ? 2 : DT;
            a *= scale;
            c *= scale;
            if (t.weight) {
                a *= load_any(t.weight, wt, at0) + p.offset;
                c *= load_any(t.weight, wt, at1) + p.offset;
            }
        }
        if (i < p.pairs) {
            float sine, cosine;
            pair_turn(p, pos, i, sine, cosine);
            turn(a, c, sine, cosine);
        }
        store_any(t.out, DT, to + at0, a);
        store_any(t.out, DT, to + at1, c);
    }
}

}  // namespace

#define DFQ_ROPE_KERNELS(op, norm, name, dt)                                                \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void dfq_##op##_halves_##name(  \
        RopeParams p) {                                                                     \
        rotate_heads<dt, norm, false>(p);                                                   \
    }                                                                                       \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void dfq_##op##_pairs_##name(   \
        RopeParams p) {                                                                     \
        rotate_heads<dt, norm, true>(p);                                                    \
    }                                                                                       \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void dfq_##op##_any_##name(     \
        RopeParams p) {                                                                     \
        rotate_any<dt, norm>(p);                                                            \
    }
#define DFQ_ROPE_TYPES(op, norm)          \
    DFQ_ROPE_KERNELS(op, norm, bf16, 0)   \
    DFQ_ROPE_KERNELS(op, norm, f16, 1)    \
    DFQ_ROPE_KERNELS(op, norm, f32, 2)
DFQ_ROPE_TYPES(rope, kAlone)
DFQ_ROPE_TYPES(norm_rope, kNorm)
DFQ_ROPE_TYPES(norm_small_rope, kNormSmall)
