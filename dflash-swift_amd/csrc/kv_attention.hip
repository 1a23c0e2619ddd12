/*
 * kv_attention.hip -- gfx950 attention of a verify block's rows over quantised K and V, built
 * once per head width (DFQ_HEAD_DIM).
 *
 * With token t's K and V values s c + b (c the code, s and b its group's scale and bias) and a
 * row's query q:
 *   z_t = scale sum_g [ s_tg (q_g . c_tg) + b_tg sum(q_g) ]
 *   y   = sum_t h_tg [ c_t + b_tg / s_tg ] / sum_t p_t,   h_tg = p_t s_tg,
 *   p_t = 2^(z_t log2 e - M)
 * so that both products run on the codes themselves.  K's scales and biases meet the sums in fp32;
 * the weights h are rounded to fp16, and V's ratios b / s to 22 bits (see stage_scales).
 *
 * A workgroup takes a block of 16 or 32 rows of one head (a verify block's rows and the query heads
 * of a K/V head together; over a shared prefix, those of all sequences) and a range of tokens, 32
 * a wave at a time: the scores of a tile of 32 tokens leave the matrix cores in the layout in which
 * the weights go back into them, so that a wave needs no other wave until its range is over.  The
 * codes go from memory straight into LDS.  The ranges' parts meet in a second kernel (join), where
 * there is more than one.
 *
 * What bounds it.  Long caches and shared prefixes: issue of vector instructions.  A tile of 32
 * rows and 32 tokens with heads of 128 is some 435 of them at 4.3 cycles and 40 matrix steps at 16
 * on each SIMD; it takes 2700 cycles.  16 sequences of 8 rows of 40 heads over 16384 shared tokens
 * (44 GFLOP) 100 us, 440 TFLOP/s; 8 rows over 32776 tokens of their own 28 us, 38 MB at 1.4 TB/s.
 * Few tokens: a launch and code that each CU runs once (up to 128 tokens 6.5 us with heads of 64,
 * 7.5 of 128, 10.8 of 256; where a join follows, 8.8, 10.4 and 14).
 *
 * Measured and not taken: unpacking codes once a workgroup into fp16 tiles in LDS for up to 64 rows
 * (half the vector instructions, but a barrier a round and two waves a SIMD: 112 us where this took
 * 111); three and four row tiles (103 and 137 KB of LDS at heads of 128: a workgroup a CU).
 */
#include <type_traits>

#include "kv_params.h"
#include "qmm_device.h"

namespace {

constexpr int kDim = DFQ_HEAD_DIM;
constexpr int kWaves = DFQ_KV_THREADS / 64;
constexpr float kNever = -__FLT_MAX__;   /* the offset of a row that has seen nothing */

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

/* fp16 operands hold codes as the denormal numbers c 2^-24 (or 16 c 2^-24 where a code stays in
 * the upper nibble of a byte), which the matrix cores multiply exactly: a code costs a mask, and
 * no conversion.  The sums are scaled back by 2^24. */
constexpr float kUnit = 16777216.0f;
/* Scores are kept 2^-8 of what the scaled queries give, so that a query's sums fit fp16. */
constexpr float kScaleUnit = kUnit / 256.0f;
/* K's scales carry it; 4-bit codes stand in the operands sixteenfold. */
template <int BITS>
constexpr float kKScaleOf = BITS == 4 ? kScaleUnit / 16.0f : kScaleUnit;
constexpr float kMost = 3.38e38f;     /* finite numbers below it stay so in bf16 */

__device__ __forceinline__ f16x8_t as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    u32x4_t v = {a, b, c, d};
    return __builtin_bit_cast(f16x8_t, v);
}

__device__ __forceinline__ f32x4_t mfma(f16x8_t a, f16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

/* A condition whose code is kept out of the others' way. */
__device__ __forceinline__ bool rarely(bool b) { return __builtin_expect(b, false); }

/* A pointer that is the same in every lane, in scalar registers. */
__device__ __forceinline__ const char* uniform(const void* p) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
    return (const char*)(uintptr_t)((uint64_t)hi << 32 | lo);
}

/* Orders a wave's own LDS writes and reads. */
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

/* log of 2^top sum. */
__device__ __forceinline__ float log_sum(float top, float sum) {
    return sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * 0.693147180559945309f;
}

/* n / by. */
__device__ __forceinline__ int divided(int n, const Divisor& d) {
    return (int)((__umulhi((uint32_t)n, d.mul) + (uint32_t)n) >> d.shift);
}

/* The largest and the sum of the L neighbouring lanes around each (4, 8, 16 or 32). */
template <int L>
__device__ __forceinline__ float largest_of(float v) {
    v = __uint_as_float(group_of<L < 16 ? L : 16>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
    return L == 32 ? fmaxf(v, __shfl_xor(v, 16)) : v;
}
template <int L>
__device__ __forceinline__ float sum_of(float v) {
    return __uint_as_float(group_of<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

/* v combined with the lanes 16, 32 and 48 on, in each: rows of 16 lanes, then halves of the wave are
 * exchanged between two copies.  The swaps carry their own wait states on both sides. */
template <typename Op>
__device__ __forceinline__ float quarters(float v, Op op) {
    float a = v, b = v;
    __asm__ volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 4" : "+v"(a), "+v"(b));
    a = b = op(a, b);
    __asm__ volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 4" : "+v"(a), "+v"(b));
    return op(a, b);
}
__device__ __forceinline__ float quarters_sum(float v) {
    return quarters(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float quarters_largest(float v) {
    return quarters(v, [](float a, float b) { return fmaxf(a, b); });
}

/* Everything of one (head, row block, token range) of a launch. */
struct Job {
    const char *k, *v;          /* codes of the slot-and-head's first token        */
    const uint16_t *scale, *bias;   /* this lane's (K's or V's) from there         */
    int64_t slot;       /* part slot of the range                                 */
    int row0, nrows;    /* rows of this block, among the head's batch*rows*group   */
    int t0, t1;         /* the range                                              */
    int clear;          /* tokens before it are seen by every row                 */
    int first, n;       /* own caches: position of block row 0, tokens; else n     */
};

template <int BITS, int GS, bool F16, int RT>
struct Attention {
    static constexpr int kGroups = kDim / GS;
    static constexpr int kSteps = GS / 32;               /* matrix steps of a group    */
    static constexpr int kChunk = kSteps < 2 ? 1 : 2;    /* steps read from LDS at once */
    static constexpr int kChunks = kGroups * kSteps / kChunk;
    static constexpr int kWords = kChunk * BITS / 4;     /* a lane's words of them     */
    static constexpr int kRowBytes = kDim * BITS / 8;
    static constexpr int kTiles = GS / 16;               /* V column tiles of a group  */
    static constexpr int kVBytes = GS * BITS / 128;      /* a lane's bytes of a group  */
    static constexpr int kTileBytes = 32 * kRowBytes;    /* codes of 32 tokens         */
    static constexpr int kLoads = kTileBytes / 1024;     /* wave loads of them         */
    /* K and V tiles in LDS: two of each, or one where two would leave a CU fewer workgroups.  One
     * row of 16 sequences over 8192 tokens 34.9 us with one, 32.7 with two; at rows of 128 bytes,
     * 16 rows of 16 heads of 256 over 16000 tokens 26.1 with one, 31.0 with two. */
    static constexpr int kBufs = kRowBytes <= 64 ? 2 : 1;
    static constexpr float kCentre = BITS == 4 ? 8.0f : 128.0f;
    static constexpr int kRows = 16 * RT;
    using half8_t = std::conditional_t<F16, f16x8_t, bf16x8_t>;

    /* A wave's tile of scales and biases, by token.  K's biases stay as they are stored: they
     * meet the queries' sums in one matrix product. */
    struct Scales {
        union {
            float k[kGroups][32];              /* K scales * kScaleUnit                     */
            uint16_t far[2 * kGroups][32];     /* later: V's far middles in two bf16 parts  */
        };
        float v[kGroups][32];                  /* V scales                                  */
        float size[32];                        /* log2 of a token's largest V scale         */
        uint16_t kb[32 * kGroups];             /* K biases                                  */
        uint16_t ratio[2 * kGroups][32];       /* what is added to V's codes, in two fp16 parts */
    };

    /* Lanes 0..31 load K's scale and bias of token t + lane, lanes 32..63 V's of t + lane - 32. */
    struct TokenScales {
        uint16_t s[kGroups], b[kGroups];
    };
    static __device__ __forceinline__ void load_scales(const Job& job, int t, int lane,
                                                       TokenScales& out) {
        int tok = t + (lane & 31);
        if (tok >= job.n) tok = job.n - 1;
        __builtin_memcpy(out.s, job.scale + (int64_t)tok * kGroups, 2 * kGroups);
        __builtin_memcpy(out.b, job.bias + (int64_t)tok * kGroups, 2 * kGroups);
    }

    struct Rows {
        f32x4_t o[RT][kDim / 16];      /* rows 4 c + r of a tile, one column a lane        */
        float off[RT], sum[RT];        /* a row's offset M; its lane's part of sum p       */
        f32x4_t bias[RT];              /* what the biases add, column 2 g + part           */
        float unit[RT];                /* score units to log2                              */
        float from[RT];                /* what a row's scores are counted from, mostly 0   */
        bool moved;                    /* whether any is not                               */
        uint64_t apart;                /* what even_groups took from a group's scales, log2, a
                                        * byte each                                        */
        uint32_t mask[RT];             /* block rows that the row sees                     */
    };

    static __device__ __forceinline__ bool sees(const Job& job, uint32_t mask, int tok) {
        return tok < job.clear || (tok < job.n && (mask >> (tok - job.first) & 1));
    }

    /* Where the groups' V scales are 2^8 and more apart, they are brought to one size, that of the
     * smallest group: h of one group would be denormal beside another's 2^20 times as large.  A
     * group's size is the mean exponent of its scales over the wave's first tile, of the tokens
     * that all rows see (what a row does not see may not move its roundings); zeros count as their
     * token's largest. */
    static constexpr uint32_t kApart = 8;
    static __device__ __forceinline__ uint64_t even_groups(const Job& job, int t, int lane,
                                                           const Scales& sc, const Rows& st) {
        uint32_t all = ~0u;
        if (t + 32 > job.clear) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                if (rt * 16 + (lane & 15) < job.nrows) all &= st.mask[rt];
            all = group_of<16>(all, [](uint32_t a, uint32_t b) { return a & b; });
        }
        const bool counts = lane >= 32 && sees(job, all, t + (lane & 31));
        const int n = max(__popcll(__ballot(counts)), 1);
        const auto exponent = [&](int g) { return __float_as_uint(sc.v[g][lane & 31]) >> 23 & 255u; };
        uint32_t most = 0;
#pragma unroll 1
        for (int g = 0; g < kGroups; ++g) most = max(most, exponent(g));
        uint64_t means = 0;   /* a byte each */
        uint32_t least = 255;
#pragma unroll 1
        for (int g = 0; g < kGroups; ++g) {
            const uint32_t e = exponent(g);
            const uint32_t v = group_of<16>(counts ? e ? e : most : 0u,
                                            [](uint32_t x, uint32_t y) { return x + y; });
            const uint32_t sum = __builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48);
            const uint32_t mean = __builtin_amdgcn_readfirstlane(sum / n);
            means |= (uint64_t)mean << 8 * g;
            least = min(least, mean);
        }
        uint64_t apart = 0;
#pragma unroll 1
        for (int g = 0; g < kGroups; ++g) {
            const uint32_t by = (uint32_t)(means >> 8 * g & 255u) - least;
            if (by >= kApart) apart |= (uint64_t)min(by, 60u) << 8 * g;
        }
        return apart;
    }

    /* What V's biases add.  The matrix cores take a token's weight and scale as h = p s rounded to
     * fp16, and h meets the codes and, in the same form, the ratio r = b / s: h (c + r) is off by
     * what h is, 2^-12 of the value itself.  With the bias met by p instead, codes and bias cancel
     * with different roundings where a group's values lie far from its middle (a channel that
     * stands apart from its group's others): 64 tokens with one of 64 channels off by 16 of their
     * 0.3, the others' errors were 9 (8 bits, 25) times the output's own rounding, and with p in
     * 16 bits still 2.  r comes in two fp16 parts, 22 bits.
     * Where the middle b + centre s is more than 128 times the codes' half range (or s is 0), r
     * would pass fp16.  There r is -centre, codes count from the middle, which they change little,
     * and the far middle meets p itself, both in two bf16 parts (16 bits).  The offset of a row's
     * weights keeps p m below 2^35 as it keeps h below 2^15: for it, a far middle counts as a scale
     * of 2^-20 of it.
     * A V group whose scale or bias is not finite (or the middle of its range past bf16) counts as
     * a NaN scale and no bias: the rows that see it get NaN, and the others, whose weight is 0,
     * nothing. */
    struct Far {
        uint32_t m[kGroups];   /* lanes 32..63: a token's far middles, high part below, or 0 */
        bool any, nan;         /* whether the tile has such a middle, a NaN scale */
    };
    static __device__ __forceinline__ void put_ratio(Scales& sc, int g, int tok, float r) {
        const _Float16 hi = (_Float16)r, lo = (_Float16)(r - (float)hi);
        sc.ratio[2 * g][tok] = __builtin_bit_cast(uint16_t, hi);
        sc.ratio[2 * g + 1][tok] = __builtin_bit_cast(uint16_t, lo);
    }
    static __device__ __forceinline__ void stage_scales(const Job& job, int t, bool first,
                                                        const TokenScales& in, int lane,
                                                        Scales& sc, Far& far, Rows& st) {
        const int tok = lane & 31;
        bool plain = true;   /* near middles, scales of one size */
        wave_order();
        if (lane < 32) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
                sc.k[g][tok] = elem_to_f32<F16>(in.s[g]) * kKScaleOf<BITS>;
            __builtin_memcpy(__builtin_assume_aligned(sc.kb + tok * kGroups, 2 * kGroups), in.b,
                             2 * kGroups);
        } else {
            float size = 0.0f, least = __builtin_inff();
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const float s = elem_to_f32<F16>(in.s[g]), b = elem_to_f32<F16>(in.b[g]);
                plain &= is_near(s, b);
                size = fmaxf(size, fabsf(s));
                least = fminf(least, fabsf(s));
                sc.v[g][tok] = s;
                put_ratio(sc, g, tok, b * __builtin_amdgcn_rcpf(s));
            }
            plain &= size < least * (float)(1 << (kApart - 1));
            sc.size[tok] = log2_above(size);
        }
        far.any = far.nan = false;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) far.m[g] = 0;
        if (rarely(!__all(plain) || st.apart)) {
            bool nan = false;
            uint32_t seen = 0;
            if (kGroups > 1 && first) {
                wave_order();
                st.apart = even_groups(job, t, lane, sc, st);
            }
            if (lane >= 32) {
                float size = 0.0f;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    const float s = elem_to_f32<F16>(in.s[g]), b = elem_to_f32<F16>(in.b[g]);
                    const float mid = fmaf(kCentre, s, b);
                    const bool fine = fabsf(s) < __builtin_inff() && fabsf(mid) < kMost;
                    const int by = (int)(st.apart >> 8 * g & 255u);
                    sc.v[g][tok] = fine ? ldexpf(s, -by) : __builtin_nanf("");
                    if (fine) size = fmaxf(size, ldexpf(fabsf(s), -by));
                    if (!is_near(s, b)) {
                        put_ratio(sc, g, tok, -kCentre);
                        const float m = fine ? ldexpf(mid, -by) : 0.0f;
                        size = fmaxf(size, fabsf(m) * 0x1p-20f);
                        const __bf16 top = (__bf16)m, rest = (__bf16)(m - (float)top);
                        far.m[g] = __builtin_bit_cast(uint16_t, top) |
                                   (uint32_t)__builtin_bit_cast(uint16_t, rest) << 16;
                    }
                    seen |= far.m[g];
                    nan |= !fine;
                }
                sc.size[tok] = log2_above(size);
            }
            far.any = __any(seen != 0);
            far.nan = __any(nan);
        }
        wave_order();
    }
    /* log2 of a scale, rounded up to a whole number; the least is -64, so that sums of weights stay
     * finite where the scales are 0. */
    static __device__ __forceinline__ float log2_above(float size) {
        return fmaxf((float)((int)(__float_as_uint(size) >> 23) - 126), -64.0f);
    }
    /* Whether a group's middle is within 128 times its codes' half range: false where the scale is 0
     * (or under 2^-100, whose reciprocal may not be finite), infinite or NaN. */
    static __device__ __forceinline__ bool is_near(float s, float b) {
        return fabsf(fmaf(kCentre, s, b)) < fmaf(128.0f * kCentre, fabsf(s), -0x1p-100f);
    }

    /* A lane's 8 tokens of one array and group: 4 c + 0..3 of each half of the tile. */
    static __device__ __forceinline__ void tokens_of(const float* a, int c, float (&out)[8]) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const f32x4_t v = *(const f32x4_t*)(a + 16 * tt + 4 * c);
#pragma unroll
            for (int r = 0; r < 4; ++r) out[4 * tt + r] = v[r];
        }
    }

    /* The same of what a lane's column (2 g + part) of a product with the biases takes. */
    static __device__ __forceinline__ void parts_of(const uint16_t (*a)[32], int lane,
                                                    uint32_t (&out)[4]) {
        const uint16_t* p = a[lane & 15 & (2 * kGroups - 1)] + 4 * (lane >> 4);
        __builtin_memcpy(out, __builtin_assume_aligned(p, 8), 8);
        __builtin_memcpy(out + 2, __builtin_assume_aligned(p + 16, 8), 8);
    }

    /* Codes of tokens t .. t+31 straight into LDS, a row after the other as in memory, each row's
     * 16-byte pieces exchanged by turn(): rows that one read instruction takes together then lie
     * in different banks.  The instruction takes its LDS address from M0 and puts lane l's 16
     * bytes 16 l behind it, so the exchange is made in the address that a lane loads from; the
     * compiler does not see the loads, and loaded() waits for them.  Tokens past the last are the
     * last. */
    static constexpr int kPieces = kRowBytes / 16;
    static __device__ __forceinline__ int turn(int row) {
        if constexpr (kPieces <= 4) return row / (8 / kPieces) % kPieces * 16;
        else return row % 8 * 16;
    }
    static __device__ __forceinline__ void load_codes(const char* base, int n, int t, int lane,
                                                      char* to) {
        const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)to;
        const int row = lane / kPieces, piece = lane % kPieces * 16;
        const bool whole = t + 32 <= n;
        uint32_t at = (uint32_t)(t + row) * kRowBytes + (piece ^ turn(row));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            constexpr int kEach = 64 / kPieces;   /* rows a load */
            uint32_t a = (kEach % 8 ? at ^ (uint32_t)(i * kEach % 8 * 16) : at) + i * 1024;
            if (!whole) {
                const int tok = t + i * kEach + row;
                a -= (uint32_t)(tok < n ? 0 : tok - n + 1) * kRowBytes;
            }
            uint32_t m0;   /* the compiler's own, which no clobber list can name */
            __asm__ volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
                             "global_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                             : "=&s"(m0)
                             : "v"(a), "s"(base),
                               "s"(__builtin_amdgcn_readfirstlane(lds + i * 1024))
                             : "memory");
        }
    }

    /* Waits until no more than LEFT of the wave's loads are under way. */
    template <int LEFT>
    static __device__ __forceinline__ void loaded() {
        __asm__ volatile("s_waitcnt vmcnt(%0)" :: "n"(LEFT) : "memory");
    }
    /* Waits for the wave's LDS reads: what they read may be written over. */
    static __device__ __forceinline__ void read_done() {
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }

    /* 8 codes of step st of a chunk.  4 bits: the word's nibbles in the order 0 4 1 5 2 6 3 7, all
     * times 16; 8 bits: in order.  The queries are laid out to match.  The matrix cores line up the
     * products of a sum by their operands' exponents, which for denormal codes say nothing of
     * their size: with nibbles left in the low four bits, where they cost no shift, sums kept
     * some 2^-20 of their size, and a log-sum of 18 tokens was 1.2e-6 off. */
    static __device__ __forceinline__ f16x8_t k_operand(const uint32_t (&w)[kWords], int st) {
        if constexpr (BITS == 4) {
            constexpr uint32_t kMid = 0x00f000f0u;
            const uint32_t a = w[st];
            return as_f16x8(a << 4 & kMid, a & kMid, a >> 4 & kMid, a >> 8 & kMid);
        } else {
            const uint32_t a = w[2 * st], b = w[2 * st + 1];
            return as_f16x8(__builtin_amdgcn_perm(0u, a, 0x0c010c00u),
                            __builtin_amdgcn_perm(0u, a, 0x0c030c02u),
                            __builtin_amdgcn_perm(0u, b, 0x0c010c00u),
                            __builtin_amdgcn_perm(0u, b, 0x0c030c02u));
        }
    }

    /* Whether column tile i holds its codes times 16.  V's others stay in the low nibble, where a
     * sum keeps 2^-21 of the group's extent: under the outputs' rounding, but for a channel that
     * stands still 2^6 (fp16; bf16 2^9) under its group's others (4096 tokens, 4 bits, one channel
     * off by 16 of 0.3: 0.9 of the fp16 rounding more, the other tiles' channels 0.2). */
    static constexpr __device__ bool odd_tile(int i) { return BITS == 4 && (i & 1); }

    /* What a lane reads for one chunk of steps: its quarter's 8-channel pieces of tokens l % 16
     * and l % 16 + 16, and the queries'. */
    struct Chunk {
        uint32_t w[2][kWords];
        f16x8_t q[RT][kChunk];
    };
    static __device__ __forceinline__ void read_chunk(const char* tile, const f16x8_t* qlds, int ch,
                                                      int lane, Chunk& out) {
        constexpr int kPer = kSteps / kChunk;   /* chunks of a group */
        const int g = ch / kPer, part = ch % kPer, row = lane & 15;
        const int at = ((lane >> 4) * kPer + part) * kWords * 4;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const char* p = tile + ((row + 16 * tt) * kRowBytes +
                                    (at ^ turn(row) ^ (g * (GS * BITS / 8))));
            __builtin_memcpy(out.w[tt], __builtin_assume_aligned(p, kWords * 4), kWords * 4);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int s = 0; s < kChunk; ++s)
                out.q[rt][s] = qlds[(rt * (kDim / 32) + ch * kChunk + s) * 64 + lane];
    }

    /* What a lane reads for the values of group g: channels (GS / 16) (l % 16) .. of the 8 tokens
     * whose scores it also holds, 4 c + r and 16 + 4 c + r, and the tokens' scales. */
    struct Values {
        uint32_t w[8][kVBytes < 4 ? 1 : kVBytes / 4];
        float s[8];
    };
    static __device__ __forceinline__ void read_values(const char* tile, const Scales& sc, int g,
                                                       int lane, Values& out) {
        const int c = lane >> 4, at = (lane & 15) * kVBytes ^ (g * (GS * BITS / 8));
        tokens_of(sc.v[g], c, out.s);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = 4 * c + (j & 3);
            const char* p = tile + (row * kRowBytes + (at ^ turn(row))) + (j >> 2) * 16 * kRowBytes;
            if constexpr (kVBytes == 1) out.w[j][0] = *(const uint8_t*)p;
            else if constexpr (kVBytes == 2) out.w[j][0] = *(const uint16_t*)p;
            else __builtin_memcpy(out.w[j], __builtin_assume_aligned(p, kVBytes), kVBytes);
        }
    }
    static __device__ __forceinline__ void v_operands(const Values& v, f16x8_t (&out)[kTiles]) {
        uint32_t o[kTiles][4];
#pragma unroll
        for (int jp = 0; jp < 4; ++jp) {
            const auto &a = v.w[2 * jp], &b = v.w[2 * jp + 1];
            if constexpr (BITS == 8 && kVBytes >= 4) {
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
                    o[i][jp] = __builtin_amdgcn_perm(b[i / 4], a[i / 4],
                                                     0x0c000c00u | (4 + (i & 3)) << 16 | (i & 3));
            } else {
                uint32_t pair[2];   /* two tokens' next 16 bits of codes */
                pair[0] = __builtin_amdgcn_perm(b[0], a[0], 0x05040100u);
                pair[1] = kVBytes == 4 ? __builtin_amdgcn_perm(b[0], a[0], 0x07060302u) : 0;
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    if constexpr (BITS == 8) {
                        o[i][jp] = pair[0] >> 8 * i & 0x00ff00ffu;
                    } else {
                        const uint32_t x = pair[i >> 2] >> (i & 2 ? 8 : 0);
                        o[i][jp] = x & (i & 1 ? 0x00f000f0u : 0x000f000fu);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) out[i] = as_f16x8(o[i][0], o[i][1], o[i][2], o[i][3]);
    }

    /* One tile of 32 tokens: scores from k, then the next tile's K, then the values. */
    template <bool MASKED>
    static __device__ __forceinline__ void scores(const Job& job, int t, int lane,
                                                  const char* k, const Scales& sc,
                                                  const f16x8_t* qlds, const half8_t* qsums,
                                                  const Rows& st, float (&z)[RT][8]) {
        const int c = lane >> 4;
        /* what is read from LDS is read one chunk ahead of its use */
        uint32_t kb[2][4] = {};
        half8_t qs[RT];
        Chunk in;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
            __builtin_memcpy(kb[tt], __builtin_assume_aligned(
                sc.kb + ((lane & 15) + 16 * tt) * kGroups, 2 * kGroups), 2 * kGroups);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) qs[rt] = qsums[rt * 64 + lane];
        read_chunk(k, qlds, 0, lane, in);
        __builtin_amdgcn_sched_barrier(0);
        /* sum_g b_g sum(q_g): the sums come in three 16-bit parts, one a quarter of the lanes */
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const u32x4_t v = {kb[tt][0], kb[tt][1], kb[tt][2], kb[tt][3]};
                const f32x4_t b = mfma(__builtin_bit_cast(half8_t, v), qs[rt],
                                       f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int r = 0; r < 4; ++r) z[rt][4 * tt + r] = b[r];
            }
        f32x4_t acc[RT][2];
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
            constexpr int kPer = kSteps / kChunk;
            if (ch % kPer == 0)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    for (int tt = 0; tt < 2; ++tt) acc[rt][tt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int st = 0; st < kChunk; ++st) {
                const f16x8_t a0 = k_operand(in.w[0], st), a1 = k_operand(in.w[1], st);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    acc[rt][0] = mfma(a0, in.q[rt][st], acc[rt][0]);
                    acc[rt][1] = mfma(a1, in.q[rt][st], acc[rt][1]);
                }
            }
            const int g = ch / kPer;
            const bool last = ch % kPer == kPer - 1;
            float s[8];
            if (last) tokens_of(sc.k[g], c, s);
            if (ch + 1 < kChunks) read_chunk(k, qlds, ch + 1, lane, in);
            __builtin_amdgcn_sched_barrier(0);
            if (last)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        z[rt][j] = fmaf(s[j], acc[rt][j >> 2][j & 3], z[rt][j]);
        }
        if constexpr (MASKED) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int tok = t + 16 * (j >> 2) + 4 * c + (j & 3);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (!sees(job, st.mask[rt], tok)) z[rt][j] = -__builtin_inff();
            }
        }
    }

    static __device__ __forceinline__ float largest_product(const float (&z)[8], float unit,
                                                            const float (&size)[8]) {
        float top = fmaf(z[0], unit, size[0]);
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, fmaf(z[j], unit, size[j]));
        return top;
    }

    /* Softmax weights of the tile's scores and their product with V.  A row's offset M is kept
     * so that p s stays below 2^15: p s is rounded to fp16 for the matrix cores, whose 2^-14
     * least normal number then lies 2^-29 under it.  M rises only when a tile would pass 2^15,
     * to where its largest is 2^11.  It goes by each token's own score and scale: a token of huge
     * values and no weight does not move it.
     * Where M would pass 2^10 in size, the row's scores are counted from the tile's largest, and M
     * with them: an M of 2^26 could not be placed within the 2^4 that p s has above 2^11, and past
     * that p would be infinite or 0 throughout. */
    template <bool MASKED>
    static __device__ __forceinline__ void weigh(const Job& job, int t, int lane,
                                                 const char* v, Scales& sc, const Far& far,
                                                 Rows& st, float (&z)[RT][8]) {
        const int c = lane >> 4;
        Values in;
        float size[8];
        uint32_t ratio[4];
        tokens_of(sc.size, c, size);
        parts_of(sc.ratio, lane, ratio);
        read_values(v, sc, 0, lane, in);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (rarely(st.moved))
#pragma unroll
                for (int j = 0; j < 8; ++j) z[rt][j] -= st.from[rt];
            float top = largest_product(z[rt], st.unit[rt], size);
            if (__any(top > st.off[rt] + 15.0f)) {
                top = quarters_largest(top);
                float off = st.off[rt], next = fmaxf(off, top - 11.0f);
                const bool move = next > off && fabsf(next) > 0x1p10f;
                if (rarely(__any(move))) {
                    float by = z[rt][0];
#pragma unroll
                    for (int j = 1; j < 8; ++j) by = fmaxf(by, z[rt][j]);
                    by = quarters_largest(by);
                    by = move && fabsf(by) < __builtin_inff() ? by : 0.0f;
                    st.from[rt] += by;
                    st.moved = true;
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[rt][j] -= by;
                    top = quarters_largest(largest_product(z[rt], st.unit[rt], size));
                    off = off == kNever ? off : fmaf(-by, st.unit[rt], off);
                    next = fmaxf(off, top - 11.0f);
                }
                const float keep = next == off ? 1.0f : exp2f(off - next);
                st.off[rt] = next;
                st.sum[rt] *= keep;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = __shfl(keep, 4 * c + r);
                    st.bias[rt][r] *= f;
#pragma unroll
                    for (int i = 0; i < kDim / 16; ++i) st.o[rt][i][r] *= f;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z[rt][j] = __builtin_amdgcn_exp2f(fmaf(z[rt][j], st.unit[rt], -st.off[rt]));
                st.sum[rt] += z[rt][j];
            }
        }
        if (rarely(far.any)) {
            /* sum p m of all groups at once, p and m in two bf16 parts each */
            wave_order();
            if (lane >= 32)
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    sc.far[2 * g][lane & 31] = (uint16_t)far.m[g];
                    sc.far[2 * g + 1][lane & 31] = (uint16_t)(far.m[g] >> 16);
                }
            wave_order();
            uint32_t m[4];
            parts_of(sc.far, lane, m);
            const u32x4_t b = {m[0], m[1], m[2], m[3]};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                u32x4_t hi, lo;
#pragma unroll
                for (int jp = 0; jp < 4; ++jp) {
                    const f32x2_t x = {z[rt][2 * jp], z[rt][2 * jp + 1]};
                    const bf16x2_t h = __builtin_convertvector(x, bf16x2_t);
                    const f32x2_t rest = {x[0] - (float)h[0], x[1] - (float)h[1]};
                    hi[jp] = __builtin_bit_cast(uint32_t, h);
                    lo[jp] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, bf16x2_t));
                }
                st.bias[rt] = mfma(__builtin_bit_cast(bf16x8_t, hi), __builtin_bit_cast(bf16x8_t, b),
                                   st.bias[rt]);
                st.bias[rt] = mfma(__builtin_bit_cast(bf16x8_t, lo), __builtin_bit_cast(bf16x8_t, b),
                                   st.bias[rt]);
            }
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            f16x8_t w[kTiles];
            v_operands(in, w);
            float s[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] = in.s[j];
            /* the other groups' columns of the product with the ratios stay as they are */
            const bool mine = (lane & 15) >> 1 == g;
            const f16x8_t r = as_f16x8(mine ? ratio[0] : 0, mine ? ratio[1] : 0,
                                       mine ? ratio[2] : 0, mine ? ratio[3] : 0);
            __builtin_amdgcn_sched_barrier(0);
            if (g + 1 < kGroups) {
                read_values(v, sc, g + 1, lane, in);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                uint32_t ps[4];
#pragma unroll
                for (int jp = 0; jp < 4; ++jp) {
                    f32x2_t x = {z[rt][2 * jp] * s[2 * jp], z[rt][2 * jp + 1] * s[2 * jp + 1]};
                    if constexpr (MASKED) {
                        const int tok = t + 16 * (jp >> 1) + 4 * c + 2 * (jp & 1);
                        if (!sees(job, st.mask[rt], tok)) x[0] = 0.0f;
                        if (!sees(job, st.mask[rt], tok + 1)) x[1] = 0.0f;
                    }
                    ps[jp] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2_t));
                }
                f16x8_t a = as_f16x8(ps[0], ps[1], ps[2], ps[3]);
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
                    st.o[rt][g * kTiles + i] = mfma(a, w[i], st.o[rt][g * kTiles + i]);
                if (rarely(far.nan))   /* stays in its own group */
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] = a[j] == a[j] ? a[j] : (_Float16)0.0f;
                st.bias[rt] = mfma(a, r, st.bias[rt]);
            }
        }
    }

    /* LDS of a workgroup.  The waves' results meet in it when the loop is over. */
    struct Lds {
        union {
            struct {
                __attribute__((aligned(16))) char pool[kRows * kDim * 2];   /* queries */
                char k[kWaves][kBufs][kTileBytes], v[kWaves][kBufs][kTileBytes];
                Scales scales[kWaves];
                __attribute__((aligned(16))) uint16_t qsums[kRows * 4 * 8];
                uint32_t masks[kRows];
                float units[kRows];
            };
            struct {
                f32x4_t merge[kWaves][kDim / 16][RT][64];
                /* by row: offset, sum, and the two parts of what the biases add to a group */
                float offs[kWaves][kRows], sums[kWaves][kRows];
                float bias[kWaves][2 * kGroups][kRows];
                uint64_t apart[kWaves];
            };
        };
    };

    /* The block's queries into LDS, in the order of the K operands and scaled by a power of two
     * so that a row's largest element lies in [2^14, 2^15): fp16 then holds them as exactly as
     * bf16 or fp16 did, down to 2^-29 of the largest.  unit: what takes a sum over codes times
     * 2^-24 to scores in log2; qsum: the sums of a row's groups in those units. */
    static constexpr int kLanes = kDim / 8, kPass = DFQ_KV_THREADS / kLanes;
    static constexpr int kPasses = (kRows + kPass - 1) / kPass;
    struct Queries {
        u32x4_t raw[kPasses];
        uint32_t mask[kPasses];
    };
    static __device__ __forceinline__ void load_queries(const KvAttnParams& p, const Job& job,
                                                        int h, Queries& in) {
        const int piece = threadIdx.x % kLanes, group = (int)p.group.by;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int r = threadIdx.x / kLanes + i * kPass;
            in.raw[i] = u32x4_t{0, 0, 0, 0};
            in.mask[i] = 0;
            if (r < job.nrows) {
                const int row = job.row0 + r, bm = divided(row, p.group);
                in.raw[i] = *(const u32x4_any*)(p.q + bm * p.q_stride +
                                                (int64_t)(h * group + row - bm * group) * kDim +
                                                piece * 8);
                in.mask[i] = p.tree ? p.tree[bm]
                                    : (2u << (bm - divided(bm, p.rows) * (int)p.rows.by)) - 1;
            }
        }
        /* all there, before loads that the compiler does not see are under way: it would wait
         * for those too */
#pragma unroll
        for (int i = 0; i < kPasses; ++i)
            __asm__ volatile("" :: "v"(in.raw[i]), "v"(in.mask[i]) : "memory");
    }
    static __device__ __forceinline__ void stage_queries(const KvAttnParams& p, const Queries& in,
                                                         Lds& lds) {
        const int piece = threadIdx.x % kLanes;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int r = threadIdx.x / kLanes + i * kPass;
            if (r >= kRows) break;
            float f[8], top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] = elem_to_f32<F16>(j & 1 ? in.raw[i][j / 2] >> 16 : in.raw[i][j / 2] & 0xffffu);
                top = fmaxf(top, fabsf(f[j]));
            }
            top = largest_of<kLanes>(top);
            int e = (int)(__float_as_uint(top) >> 23) - 127;
            if (e < -100 || e > 127) e = e > 127 ? 127 : -100; /* a tiny or an infinite row */
            float total = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] = ldexpf(f[j], 14 - e);
                total += f[j];
            }
            total = sum_of<GS / 8>(total);
            const int g = piece / (GS / 8), u = piece % (GS / 8), c = u / kSteps, st = u % kSteps;
            if (u < 4) {
                /* 2^-8 of the group's sum in three parts of 16 bits, part i for quarter i of the
                 * lanes; quarter 3 and the elements past the groups are 0 */
                float rest = total / 256.0f;
                uint16_t part = f32_to_out<F16>(rest);
                for (int k = 0; k < u; ++k) {
                    rest -= elem_to_f32<F16>(part);
                    part = f32_to_out<F16>(rest);
                }
                uint16_t* to = lds.qsums + ((r / 16) * 64 + u * 16 + r % 16) * 8;
                to[g] = u < 3 ? part : 0;
                if (g == 0)
#pragma unroll
                    for (int j = kGroups; j < 8; ++j) to[j] = 0;
            }
            if (piece == 0) {
                /* never 0: a hidden token's -inf stays one */
                lds.units[r] = fmaxf(ldexpf(p.scale_log2e, 8 + e - 14), 0x1p-149f);
                lds.masks[r] = in.mask[i];
            }
            /* nibble order of k_operand: operand element j is channel j/2 + 4 (j%2) */
            u32x4_t o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int a = BITS == 4 ? j : 2 * j, b = BITS == 4 ? j + 4 : 2 * j + 1;
                const f32x2_t x = {f[a], f[b]};
                o[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2_t));
            }
            const int step = (r / 16) * (kDim / 32) + g * kSteps + st;
            *(u32x4_t*)(lds.pool + (step * 64 + c * 16 + r % 16) * 16) = o;
        }
    }

    static __device__ __forceinline__ void run(const KvAttnParams& p, const Job& job, int h,
                                               char* room) {
        Lds& lds = *(Lds*)room;
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        Queries queries;
        load_queries(p, job, h, queries);
        int t = job.t0 + 32 * wave;
        TokenScales scale;
        char (&k)[kBufs][kTileBytes] = lds.k[wave], (&v)[kBufs][kTileBytes] = lds.v[wave];
        if (t < job.t1) {
            load_codes(job.k, job.n, t, lane, k[0]);
            if (kBufs == 2) load_codes(job.v, job.n, t, lane, v[0]);
            load_scales(job, t, lane, scale);
        }
        stage_queries(p, queries, lds);
        __syncthreads();

        Rows st;
        st.moved = false;
        st.apart = 0;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = rt * 16 + (lane & 15);
            st.off[rt] = kNever;
            st.from[rt] = 0.0f;
            st.sum[rt] = 0.0f;
            st.unit[rt] = lds.units[r];
            st.mask[rt] = lds.masks[r];
            st.bias[rt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) st.o[rt][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }

        float z[RT][8];
        const f16x8_t* q = (const f16x8_t*)lds.pool;
        Scales& sc = lds.scales[wave];
        int buf = 0;
        while (t < job.t1) {
            const int next = t + 32 * kWaves, other = kBufs == 2 ? buf ^ 1 : 0;
            loaded<0>();
            Far far;
            stage_scales(job, t, t < job.t0 + 32 * kWaves, scale, lane, sc, far, st);
            if (next < job.t1) load_scales(job, next, lane, scale);
            if constexpr (kBufs == 2) {
                if (next < job.t1) {
                    load_codes(job.k, job.n, next, lane, k[other]);
                    load_codes(job.v, job.n, next, lane, v[other]);
                }
            } else {
                load_codes(job.v, job.n, t, lane, v[0]);
            }
            const bool masked = t + 32 > job.clear;
            if (masked) scores<true>(job, t, lane, k[buf], sc, q, (const half8_t*)lds.qsums, st, z);
            else scores<false>(job, t, lane, k[buf], sc, q, (const half8_t*)lds.qsums, st, z);
            if constexpr (kBufs == 1) {
                read_done();
                if (next < job.t1) {
                    load_codes(job.k, job.n, next, lane, k[0]);
                    loaded<kLoads>();
                } else {
                    loaded<0>();
                }
            }
            if (masked) weigh<true>(job, t, lane, v[buf], sc, far, st, z);
            else weigh<false>(job, t, lane, v[buf], sc, far, st, z);
            read_done();
            buf = other;
            t = next;
        }

        /* The waves' rows together: their outputs, offsets, sums and what the biases add meet in
         * LDS.  A wave then adds up every fourth column tile, each of its
         * lanes with the weights of its four rows. */
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) lds.merge[wave][d][rt][lane] = st.o[rt][d];
        if (lane == 0) lds.apart[wave] = st.apart;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = rt * 16 + (lane & 15), row = rt * 16 + 4 * (lane >> 4);
            const float sum = quarters_sum(st.sum[rt]);
            if (lane < 16) {
                lds.offs[wave][r] = st.off[rt] == kNever
                                        ? kNever
                                        : fmaf(st.from[rt], st.unit[rt], st.off[rt]);
                lds.sums[wave][r] = sum;
            }
            if ((lane & 15) < 2 * kGroups)
                *(f32x4_t*)&lds.bias[wave][lane & 15][row] = st.bias[rt];
        }
        __syncthreads();
        const int64_t nrows = (int64_t)p.batch * p.rows.by * p.group.by;
        const int64_t out = (job.slot * p.heads.by + h) * nrows + job.row0;
        /* one range is the whole answer */
        const bool alone = p.prefix_splits.by + p.own_splits.by == 1;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int row = rt * 16 + 4 * (lane >> 4);
            f32x4_t weight[kWaves], top, sum = {};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) weight[w] = *(const f32x4_t*)&lds.offs[w][row];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                top[i] = weight[0][i];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) top[i] = fmaxf(top[i], weight[w][i]);
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
                    weight[w][i] = __builtin_amdgcn_exp2f(weight[w][i] - top[i]);
            }
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const f32x4_t l = *(const f32x4_t*)&lds.sums[w][row];
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fmaf(l[i], weight[w][i], sum[i]);
            }
            int64_t whole[4];   /* where the row's outputs go */
            if (alone) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = job.row0 + row + i, bm = divided(at, p.group);
                    whole[i] = (int64_t)bm * p.heads.by * p.group.by + h * p.group.by +
                               (at - bm * (int)p.group.by);
                }
            }
            if (wave == 0 && (lane & 15) == 0)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (row + i >= job.nrows) continue;
                    if (!alone)
                        *(f32x2_t*)(p.part_ml + (out + row + i) * 2) = f32x2_t{top[i], sum[i]};
                    else if (p.lse)
                        p.lse[whole[i]] = log_sum(top[i], sum[i]);
                }
#pragma unroll 1
            for (int d = wave; d < kDim / 16; d += kWaves) {
                const int g = d / kTiles;
                const float back = odd_tile(d % kTiles) ? kUnit / 16.0f : kUnit;
                f32x4_t y = {};
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const f32x4_t x = lds.merge[w][d][rt][lane];
                    const f32x4_t bias = *(const f32x4_t*)&lds.bias[w][2 * g][row] +
                                         *(const f32x4_t*)&lds.bias[w][2 * g + 1][row];
                    const int by = (int)(lds.apart[w] >> 8 * g & 255u);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[i] = fmaf(ldexpf(fmaf(x[i], back, bias[i]), by), weight[w][i], y[i]);
                }
                if (alone) {
                    const int channel = g * GS + (lane & 15) * kTiles + d % kTiles;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (row + i < job.nrows)
                            p.y[whole[i] * kDim + channel] =
                                f32_to_out<F16>(sum[i] == 0.0f ? 0.0f : y[i] / sum[i]);
                    continue;
                }
                float* to = p.part_o + (out + row) * kDim + d * 16 + (lane & 15);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (row + i < job.nrows) to[i * kDim] = y[i];
            }
        }
    }
};

/* A workgroup of a launch whose row blocks have up to RT tiles: its job, and the code for the
 * tiles that the job has. */
template <int BITS, int GS, bool F16, int RT>
__device__ __forceinline__ void attention(const KvAttnParams& p) {
    using Most = Attention<BITS, GS, F16, RT>;
    constexpr int kRows = Most::kRows, kRowBytes = Most::kRowBytes, kGroups = Most::kGroups;
    __shared__ __attribute__((aligned(16))) char lds[sizeof(typename Most::Lds)];
    const int lane = threadIdx.x % 64;

    /* the job: heads go fastest, so that with 8 of them an XCD's L2 serves one */
    Job job;
    int i = divided(blockIdx.x, p.heads);
    const int h = (int)(blockIdx.x - i * p.heads.by);
    const int seq_rows = (int)(p.rows.by * p.group.by);
    int range, block;
    Divisor ranges;
    int64_t token0;   /* index of the slot-and-head's first token in the arrays */
    KvArrays jk, jv;
    const int prefix_jobs = (int)(p.prefix_splits.by * p.prefix_blocks.by);
    if (i < prefix_jobs) {
        range = divided(i, p.prefix_blocks);
        block = i - range * (int)p.prefix_blocks.by;
        ranges = p.prefix_splits;
        jk = p.prefix[0];
        jv = p.prefix[1];
        token0 = (int64_t)h * p.prefix_capacity;
        job.slot = range;
        job.row0 = block * kRows;
        job.nrows = p.batch * seq_rows - job.row0;
        job.n = job.clear = job.first = p.prefix_length;
    } else {
        i -= prefix_jobs;
        const int b = divided(i, p.own_jobs);
        i -= b * (int)p.own_jobs.by;
        range = divided(i, p.own_blocks);
        block = i - range * (int)p.own_blocks.by;
        ranges = p.own_splits;
        jk = p.own[0];
        jv = p.own[1];
        token0 = ((int64_t)b * p.heads.by + h) * p.own_capacity;
        job.slot = (int)p.prefix_splits.by + range;
        const int r0 = block * kRows;
        job.row0 = b * seq_rows + r0;
        job.nrows = seq_rows - r0;
        int n = p.lengths ? p.lengths[b] : p.max_length;
        n = n < 0 ? 0 : n > p.max_length ? p.max_length : n;
        job.n = n;
        job.first = n - (int)p.rows.by;
        job.clear = job.first < 0 ? 0 : job.first;
    }
    if (job.nrows > kRows) job.nrows = kRows;
    job.k = uniform((const char*)jk.codes + token0 * kRowBytes);
    job.v = uniform((const char*)jv.codes + token0 * kRowBytes);
    job.scale = (lane < 32 ? jk.scales : jv.scales) + token0 * kGroups;
    job.bias = (lane < 32 ? jk.biases : jv.biases) + token0 * kGroups;
    /* ranges of whole rounds of 32 tokens a wave */
    const int rounds = (job.n + 32 * kWaves - 1) / (32 * kWaves);
    const int each = divided(rounds + (int)ranges.by - 1, ranges) * 32 * kWaves;
    job.t0 = range * each < job.n ? range * each : job.n;
    job.t1 = job.t0 + each < job.n ? job.t0 + each : job.n;

    const int tiles = (job.nrows + 15) / 16;
    if constexpr (RT > 1)
        if (tiles == 1) return Attention<BITS, GS, F16, 1>::run(p, job, h, lds);
    Most::run(p, job, h, lds);
}

/* The parts of a row from all ranges, in the order of their slots: y = sum 2^(M - top) o / sum
 * 2^(M - top) l.  WAVES waves take a row's slots in turn, a lane kDim / 64 channels; the slots'
 * offsets and sums come in one load a lane (64 slots at a time), and eight slots' parts are under
 * way together, since the row waits for memory and for nothing else.  With few slots a wave has a
 * row to itself, and a workgroup four rows (40 rows of 17 slots 2.6 us, 5120 rows of 4 5.3). */
template <int GS, bool F16, int WAVES>
__device__ __forceinline__ void join(const KvAttnParams& p) {
    constexpr int kEach = kDim / 64, kAhead = 8;
    typedef float part_t __attribute__((ext_vector_type(kEach)));
    __shared__ float acc[kWaves][kDim];
    __shared__ float weight[kWaves][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, first = wave % WAVES;
    const int64_t nrows = (int64_t)p.batch * p.rows.by * p.group.by;
    const int h = blockIdx.y, slots = (int)(p.prefix_splits.by + p.own_splits.by);
    const int64_t row = (int64_t)blockIdx.x * (kWaves / WAVES) + wave / WAVES;
    if (WAVES == 1 && row >= nrows) return;
    const int64_t stride = nrows * p.heads.by, at = h * nrows + row;
    const f32x2_t* ml = (const f32x2_t*)p.part_ml + at;
    float top = kNever;
    for (int s = lane; s < slots; s += 64) top = fmaxf(top, ml[s * stride][0]);
    top = quarters_largest(largest_of<16>(top));
    float sum = 0.0f;
    part_t o = {};
    for (int s0 = 0; s0 < slots; s0 += 64) {
        const f32x2_t v = s0 + lane < slots ? ml[(s0 + lane) * stride] : f32x2_t{kNever, 0.0f};
        const float f = __builtin_amdgcn_exp2f(v[0] - top);
        sum = fmaf(v[1], f, sum);
        weight[wave][lane] = f;
        wave_order();
        const int n = slots - s0 < 64 ? slots - s0 : 64;
        for (int s = first; s < n; s += kAhead * WAVES) {
            part_t x[kAhead];
            float w[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int k = s + i * WAVES < n ? s + i * WAVES : s;
                x[i] = *(const part_t*)(p.part_o + ((s0 + k) * stride + at) * kDim + lane * kEach);
                w[i] = weight[wave][k];
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (s + i * WAVES < n) o += x[i] * w[i];
        }
        wave_order();
    }
    sum = quarters_sum(sum_of<16>(sum));
    *(part_t*)&acc[wave][lane * kEach] = o;
    if (WAVES > 1) __syncthreads();
    else wave_order();
    const int bm = divided((int)row, p.group), group = (int)p.group.by;
    const int64_t q_heads = (int64_t)p.heads.by * group;
    const int64_t head = h * group + (int)row - bm * group;
    for (int d = WAVES > 1 ? threadIdx.x : lane; d < kDim; d += 64 * WAVES) {
        /* channel d of group g is column (d % GS) / (GS / 16) of the group's tile d % (GS / 16) */
        constexpr int kTiles = GS / 16;
        const int e = (d / GS * kTiles + d % kTiles) * 16 + d % GS / kTiles;
        float v = acc[WAVES > 1 ? 0 : wave][e];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += acc[w][e];
        p.y[(bm * q_heads + head) * kDim + d] = f32_to_out<F16>(sum == 0.0f ? 0.0f : v / sum);
    }
    if (p.lse && first == 0 && lane == 0)
        p.lse[bm * q_heads + head] = log_sum(top, sum);
}

}  // namespace

/* Built for the row tiles that attention_tiles (verify_ops.cpp) asks for; per_4 and per_8 are the
 * waves that a SIMD has registers and LDS for with 4 and 8 bits.  One kernel spills at them: heads of
 * 64 with 4 bits in groups of 64, bf16, two tiles, 12 bytes a lane.  With two waves a SIMD it does not,
 * and takes 363 us for 294 (32 sequences of 8 rows of 64 heads over 30000 shared tokens); nor with the
 * rows' masks read again for each tile, 299. */
#define DFQ_ATTN(bits, gs, name, f16, rt, per_simd)                                            \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS, per_simd) void                     \
        dfq_cache_attention_b##bits##_g##gs##_##name##_r##rt(KvAttnParams p) {                 \
        attention<bits, gs, f16, rt>(p);                                                       \
    }
#define DFQ_JOIN(gs, name, f16)                                                                \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void                               \
        dfq_cache_attention_join_g##gs##_##name(KvAttnParams p) {                              \
        if (p.join_rows == 1) join<gs, f16, kWaves>(p);                                        \
        else join<gs, f16, 1>(p);                                                              \
    }
#define DFQ_FORMATS(M, gs, rt, per_4, per_8)                          \
    M(4, gs, bf16, false, rt, per_4) M(8, gs, bf16, false, rt, per_8) \
    M(4, gs, f16, true, rt, per_4) M(8, gs, f16, true, rt, per_8)
#define DFQ_JOINS(gs) DFQ_JOIN(gs, bf16, false) DFQ_JOIN(gs, f16, true)

DFQ_JOINS(32)
DFQ_JOINS(64)
#if DFQ_HEAD_DIM == 64
DFQ_FORMATS(DFQ_ATTN, 32, 1, 3, 3)
DFQ_FORMATS(DFQ_ATTN, 32, 2, 2, 2)
DFQ_FORMATS(DFQ_ATTN, 64, 1, 3, 3)
DFQ_FORMATS(DFQ_ATTN, 64, 2, 3, 3)
#elif DFQ_HEAD_DIM == 128
DFQ_JOINS(128)
DFQ_FORMATS(DFQ_ATTN, 32, 1, 3, 3)
DFQ_FORMATS(DFQ_ATTN, 32, 2, 2, 2)
DFQ_FORMATS(DFQ_ATTN, 64, 1, 3, 3)
DFQ_FORMATS(DFQ_ATTN, 64, 2, 2, 2)
DFQ_FORMATS(DFQ_ATTN, 128, 1, 3, 3)
DFQ_FORMATS(DFQ_ATTN, 128, 2, 2, 2)
#elif DFQ_HEAD_DIM == 256
DFQ_JOINS(128)
DFQ_FORMATS(DFQ_ATTN, 32, 1, 2, 1)
DFQ_FORMATS(DFQ_ATTN, 64, 1, 2, 1)
DFQ_FORMATS(DFQ_ATTN, 128, 1, 2, 2)
#else
#error "DFQ_HEAD_DIM must be 64, 128 or 256"
#endif
