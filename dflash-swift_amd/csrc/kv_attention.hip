/*
 * kv_attention.hip -- gfx950 attention of a verify block's rows over quantised K and V, built
 * once per head width (DFQ_HEAD_DIM).
 *
 * With token t's K and V values s c + b (c the code, s and b its group's scale and bias) and a
 * row's query q:
 *   z_t = scale sum_g [ s_tg (q_g . c_tg) + b_tg sum(q_g) ]
 *   y   = sum_t p_t [ s_tg c_t + b_tg ] / sum_t p_t,   p_t = 2^(z_t log2 e - M)
 * so that both products run on the codes themselves, and scales and biases meet the scores in
 * fp32: no value of the cache is rounded on the way.
 */
#include <type_traits>

#include "kv_params.h"
#include "qmm_device.h"

namespace {

constexpr int kDim = DFQ_HEAD_DIM;
constexpr int kWaves = DFQ_KV_THREADS / 64;
constexpr float kNever = -1e30f;      /* the offset of a row that has seen nothing */

typedef uint32_t u32_any __attribute__((aligned(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

/* fp16 operands hold codes as the denormal numbers c 2^-24 (or 16 c 2^-24 where a code stays in
 * the upper nibble of a byte), which the matrix cores multiply exactly: a code costs a mask, and
 * no conversion.  The sums are scaled back by 2^24. */
constexpr float kUnit = 16777216.0f;

template <bool F16>
__device__ __forceinline__ float half_of(uint32_t word, bool high) {
    if constexpr (F16)
        return (float)__builtin_bit_cast(f16x2_t, word)[high ? 1 : 0];
    else
        return __uint_as_float(high ? word & 0xffff0000u : word << 16);
}

__device__ __forceinline__ f16x8_t as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    u32x4_t v = {a, b, c, d};
    return __builtin_bit_cast(f16x8_t, v);
}

__device__ __forceinline__ f32x4_t mfma(f16x8_t a, f16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

/* Everything of one (head, row block, token range) of a launch. */
struct Job {
    const char *k, *v;          /* codes of the slot-and-head's first token        */
    const uint16_t* scale;      /* this lane's array of scales or biases from there */
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
    static constexpr int kRowBytes = kDim * BITS / 8;
    static constexpr int kKWords = GS * BITS / 128;      /* a lane's words of a group  */
    static constexpr int kTiles = GS / 16;               /* V column tiles of a group  */
    static constexpr int kVBytes = GS * BITS / 128;      /* a lane's bytes of a group  */
    static constexpr int kVWords = kVBytes < 4 ? 4 : 8 * kVBytes / 4;
    static constexpr float kCentre = BITS == 4 ? 8.0f : 128.0f;
    static constexpr int kRows = 16 * RT;

    struct KTile {
        uint32_t code[2][kGroups][kKWords];
        uint32_t scale[kGroups];   /* this lane's part of the tile's scales and biases */
    };
    struct VTile {
        uint32_t code[kGroups][kVWords];
    };
    /* A wave's tile of scales and biases in fp32, by token: K's, V's; size: a token's largest
     * finite V scale. */
    struct Scales {
        float s[4][kGroups][32];   /* K scales, K biases, V scales, V biases */
        float size[32];
    };

    /* Lane l loads array l / 16 (K scales, K biases, V scales, V biases), tokens t + 2 (l % 16)
     * and the next: 2 kGroups neighbouring 16-bit numbers. */
    template <bool TAIL>
    static __device__ __forceinline__ void load_scales(const Job& job, int t, int lane,
                                                       uint32_t (&out)[kGroups]) {
        const int tok = t + 2 * (lane & 15);
        if constexpr (!TAIL) {
            const uint16_t* p = job.scale + (int64_t)tok * kGroups;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) out[g] = *(const u32_any*)(p + 2 * g);
        } else {
            uint32_t h[2 * kGroups];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t at = tok + r < job.n ? tok + r : job.n - 1;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) h[r * kGroups + g] = job.scale[at * kGroups + g];
            }
#pragma unroll
            for (int g = 0; g < kGroups; ++g) out[g] = h[2 * g] | h[2 * g + 1] << 16;
        }
    }

    /* Orders a wave's LDS writes and reads of its own tile of scales. */
    static __device__ __forceinline__ void wave_fence() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    static __device__ __forceinline__ void stage_scales(const uint32_t (&in)[kGroups], int lane,
                                                        Scales& sc) {
        const int arr = lane >> 4, tok = 2 * (lane & 15);
        float size[2] = {0.0f, 0.0f};
        wave_fence();
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            float f[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int i = r * kGroups + g;
                f[r] = half_of<F16>(in[i >> 1], i & 1);
                const float a = fabsf(f[r]);
                size[r] = fmaxf(size[r], a < __builtin_inff() ? a : 0.0f);
            }
            *(f32x2_t*)&sc.s[arr][g][tok] = f32x2_t{f[0], f[1]};
        }
        if (arr == 2) *(f32x2_t*)&sc.size[tok] = f32x2_t{size[0], size[1]};
        wave_fence();
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

    /* K rows t .. t+31 (and all the tile's scales) as the row operand: lane l holds token l % 16 of each half and, of every
     * group, the kSteps 8-channel pieces that its quarter l / 16 multiplies. */
    template <bool TAIL>
    static __device__ __forceinline__ void load_k(const Job& job, int t, int lane, KTile& k) {
        const int row = lane & 15, c = lane >> 4;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            int tok = t + 16 * tt + row;
            if (TAIL && tok >= job.n) tok = job.n - 1;
            const uint32_t at = (uint32_t)tok * kRowBytes + c * kKWords * 4;
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
                __builtin_memcpy(k.code[tt][g],
                                 __builtin_assume_aligned(job.k + (at + g * (GS * BITS / 8)),
                                                          kKWords < 4 ? kKWords * 4 : 16),
                                 kKWords * 4);
        }
        load_scales<TAIL>(job, t, lane, k.scale);
    }

    /* V rows as the column operand: lane l holds, of every group, channels (GS / 16) (l % 16) ..
     * of the 8 tokens whose scores it also holds: t + 4 c + r and t + 16 + 4 c + r, c = l / 16. */
    template <bool TAIL>
    static __device__ __forceinline__ void load_v(const Job& job, int t, int lane, VTile& v) {
        const int col = lane & 15, c = lane >> 4;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            uint32_t at[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                int tok = t + 16 * (j >> 2) + 4 * c + (j & 3) + i;
                if (TAIL && tok >= job.n) tok = job.n - 1;
                at[i] = (uint32_t)tok * kRowBytes + col * kVBytes;
            }
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                constexpr int kStep = GS * BITS / 8;
                if constexpr (kVBytes >= 4) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        __builtin_memcpy(&v.code[g][(j + i) * (kVBytes / 4)],
                                         __builtin_assume_aligned(job.v + (at[i] + g * kStep),
                                                                  kVBytes), kVBytes);
                } else {
                    /* two tokens' halves of one register, which loads fill one by one */
                    using Piece = std::conditional_t<kVBytes == 2, uint16_t, uint8_t>;
                    u16x2_t x;
                    x[0] = *(const Piece*)(job.v + (at[0] + g * kStep));
                    x[1] = *(const Piece*)(job.v + (at[1] + g * kStep));
                    v.code[g][j >> 1] = __builtin_bit_cast(uint32_t, x);
                }
            }
        }
    }

    /* 8 codes of step st of a group.  4 bits: the word's nibbles in the order 0 4 1 5 2 6 3 7,
     * the odd ones times 16; 8 bits: in order.  The queries are laid out to match. */
    static __device__ __forceinline__ f16x8_t k_operand(const uint32_t (&w)[kKWords], int st) {
        if constexpr (BITS == 4) {
            const uint32_t a = w[st], b = a >> 8;
            return as_f16x8(a & 0x000f000fu, a & 0x00f000f0u, b & 0x000f000fu, b & 0x00f000f0u);
        } else {
            const uint32_t a = w[2 * st], b = w[2 * st + 1];
            return as_f16x8(__builtin_amdgcn_perm(0u, a, 0x0c010c00u),
                            __builtin_amdgcn_perm(0u, a, 0x0c030c02u),
                            __builtin_amdgcn_perm(0u, b, 0x0c010c00u),
                            __builtin_amdgcn_perm(0u, b, 0x0c030c02u));
        }
    }

    /* Whether column tile i holds its codes times 16. */
    static constexpr __device__ bool odd_tile(int i) { return BITS == 4 && (i & 1); }

    /* The 8 tokens' codes of channel i of a lane's group channels. */
    static __device__ __forceinline__ f16x8_t v_operand(const uint32_t (&w)[kVWords], int i) {
        uint32_t o[4];
#pragma unroll
        for (int jp = 0; jp < 4; ++jp) {
            if constexpr (BITS == 4) {
                uint32_t pair;  /* tokens 2 jp and 2 jp + 1: 16 bits of codes each */
                if constexpr (kVBytes == 4)
                    pair = __builtin_amdgcn_perm(w[2 * jp + 1], w[2 * jp],
                                                 i < 4 ? 0x05040100u : 0x07060302u);
                else
                    pair = w[jp];
                const int n = i & 3;
                const uint32_t x = n < 2 ? pair : pair >> 8;
                o[jp] = x & (n & 1 ? 0x00f000f0u : 0x000f000fu);
            } else {
                if constexpr (kVBytes == 2) {
                    o[jp] = (i ? w[jp] >> 8 : w[jp]) & 0x00ff00ffu;
                } else {
                    constexpr int kW = kVBytes / 4;
                    const uint32_t a = w[2 * jp * kW + i / 4], b = w[(2 * jp + 1) * kW + i / 4];
                    const uint32_t n = i & 3;
                    o[jp] = __builtin_amdgcn_perm(b, a, 0x0c000c00u | (4 + n) << 16 | n);
                }
            }
        }
        return as_f16x8(o[0], o[1], o[2], o[3]);
    }

    struct Rows {
        f32x4_t o[RT][kDim / 16];      /* rows 4 c + r of a tile, one column a lane        */
        float off[RT], sum[RT];        /* a row's offset M; its lane's part of sum p       */
        float code_sum[RT][kGroups];   /* its part of sum of the rounded p s               */
        float bias_sum[RT][kGroups];   /* its part of sum p (b + centre s)                 */
        float unit[RT];                /* score units to log2                              */
        float qsum[RT][kGroups];
        uint32_t mask[RT];             /* block rows that the row sees                     */
    };

    /* One tile of 32 tokens: scores from k, then the next tile's K, then the values. */
    template <bool MASKED>
    static __device__ __forceinline__ void scores(const Job& job, int t, int lane, int tiles,
                                                  const KTile& k, const Scales& sc,
                                                  const f16x8_t* qlds, const Rows& st,
                                                  float (&z)[RT][8]) {
        const int c = lane >> 4;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            f32x4_t acc[RT][2];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                for (int tt = 0; tt < 2; ++tt) acc[rt][tt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const f16x8_t a0 = k_operand(k.code[0][g], s), a1 = k_operand(k.code[1][g], s);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (rt >= tiles) break;
                    const f16x8_t q = qlds[(rt * (kDim / 32) + g * kSteps + s) * 64 + lane];
                    acc[rt][0] = mfma(a0, q, acc[rt][0]);
                    acc[rt][1] = mfma(a1, q, acc[rt][1]);
                }
            }
            float s[8], b[8];
            tokens_of(sc.s[0][g], c, s);
            tokens_of(sc.s[1][g], c, b);
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float v = g ? fmaf(b[j], st.qsum[rt][g], z[rt][j]) : b[j] * st.qsum[rt][g];
                    z[rt][j] = fmaf(s[j], acc[rt][j >> 2][j & 3], v);
                }
            if constexpr (kGroups >= 4) __builtin_amdgcn_sched_barrier(0);
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

    static __device__ __forceinline__ bool sees(const Job& job, uint32_t mask, int tok) {
        return tok < job.clear || (tok < job.n && (mask >> (tok - job.first) & 1));
    }

    /* Softmax weights of the tile's scores and their product with V.  A row's offset M is kept
     * so that p s stays below 2^15: p s is rounded to fp16 for the matrix cores, whose 2^-14
     * least normal number then lies 2^-29 under it.  M rises only when a tile would pass 2^15,
     * to where its largest is 2^11. */
    template <bool MASKED>
    static __device__ __forceinline__ void weigh(const Job& job, int t, int lane, int tiles,
                                                 const VTile& v, const Scales& sc, Rows& st,
                                                 float (&z)[RT][8]) {
        const int c = lane >> 4;
        float size[8];
        tokens_of(sc.size, c, size);
        float most = size[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) most = fmaxf(most, size[j]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (rt >= tiles) break;
            float top = z[rt][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top = fmaxf(top, z[rt][j]);
            if constexpr (MASKED) {
                most = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int tok = t + 16 * (j >> 2) + 4 * c + (j & 3);
                    if (sees(job, st.mask[rt], tok)) most = fmaxf(most, size[j]);
                }
            }
            /* log2 of the scale, rounded up to a whole number */
            const float up = fmaxf((float)((int)(__float_as_uint(most) >> 23) - 126), -40.0f);
            const float high = fmaf(top, st.unit[rt], up);
            if (__any(high > st.off[rt] + 15.0f)) {
                float all = fmaf(top, st.unit[rt], 0.0f), allup = up;
                all = fmaxf(all, __shfl_xor(all, 16));
                all = fmaxf(all, __shfl_xor(all, 32));
                allup = fmaxf(allup, __shfl_xor(allup, 16));
                allup = fmaxf(allup, __shfl_xor(allup, 32));
                const float next = fmaxf(st.off[rt], all + allup - 11.0f);
                const float keep = next == st.off[rt] ? 1.0f : exp2f(st.off[rt] - next);
                st.off[rt] = next;
                st.sum[rt] *= keep;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    st.code_sum[rt][g] *= keep;
                    st.bias_sum[rt][g] *= keep;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = __shfl(keep, 4 * c + r);
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
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            f16x8_t w[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) w[i] = v_operand(v.code[g], i);
            float s[8], b[8];
            tokens_of(sc.s[2][g], c, s);
            tokens_of(sc.s[3][g], c, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = fmaf(kCentre, s[j], b[j]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (rt >= tiles) break;
                uint32_t ps[4];
#pragma unroll
                for (int jp = 0; jp < 4; ++jp) {
                    f32x2_t x = {z[rt][2 * jp] * s[2 * jp], z[rt][2 * jp + 1] * s[2 * jp + 1]};
                    float y0 = z[rt][2 * jp] * b[2 * jp], y1 = z[rt][2 * jp + 1] * b[2 * jp + 1];
                    if constexpr (MASKED) {
                        const int tok = t + 16 * (jp >> 1) + 4 * c + 2 * (jp & 1);
                        if (!sees(job, st.mask[rt], tok)) x[0] = y0 = 0.0f;
                        if (!sees(job, st.mask[rt], tok + 1)) x[1] = y1 = 0.0f;
                    }
                    st.bias_sum[rt][g] += y0;
                    st.bias_sum[rt][g] += y1;
                    const f16x2_t h = __builtin_convertvector(x, f16x2_t);
                    ps[jp] = __builtin_bit_cast(uint32_t, h);
                    const f16x2_t one = {(_Float16)1.0f, (_Float16)1.0f};
                    st.code_sum[rt][g] = __builtin_amdgcn_fdot2(h, one, st.code_sum[rt][g], false);
                }
                const f16x8_t a = as_f16x8(ps[0], ps[1], ps[2], ps[3]);
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
                    st.o[rt][g * kTiles + i] = mfma(a, w[i], st.o[rt][g * kTiles + i]);
            }
            if constexpr (kGroups >= 4) __builtin_amdgcn_sched_barrier(0);
        }
    }

    /* The block's queries into LDS, in the order of the K operands and scaled by a power of two
     * so that a row's largest element lies in [2^14, 2^15): fp16 then holds them as exactly as
     * bf16 or fp16 did, down to 2^-29 of the largest.  unit: what takes a sum over codes times
     * 2^-24 to scores in log2; qsum: the sums of a row's groups in those units. */
    static __device__ __forceinline__ void stage_queries(const KvAttnParams& p, const Job& job,
                                                         int h, uint16_t* qlds, float* unit,
                                                         float* qsum) {
        constexpr int kLanes = kDim / 8;
        const int piece = threadIdx.x % kLanes, q_heads = p.heads * p.group;
        for (int r = threadIdx.x / kLanes; r < kRows; r += DFQ_KV_THREADS / kLanes) {
            float f[8] = {};
            if (r < job.nrows) {
                const int row = job.row0 + r, bm = row / p.group;
                const uint16_t* q = p.q + bm * p.q_stride +
                                    (int64_t)(h * p.group + row - bm * p.group) * kDim + piece * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = elem_to_f32<F16>(q[i]);
            }
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
            for (int d = 1; d < kLanes; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
            int e = (int)(__float_as_uint(top) >> 23) - 127;
            if (e < -100 || e > 127) e = e > 127 ? 127 : -100; /* a tiny or an infinite row */
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = ldexpf(f[i], 14 - e);
                total += f[i];
            }
            for (int d = 1; d < GS / 8; d *= 2) total += __shfl_xor(total, d);
            const int g = piece / (GS / 8), u = piece % (GS / 8), c = u / kSteps, st = u % kSteps;
            if (u == 0) qsum[r * kGroups + g] = total / kUnit;
            if (piece == 0) unit[r] = ldexpf(p.scale_log2e, 24 + e - 14);
            uint16_t* o = qlds + (((r / 16) * (kDim / 32) + g * kSteps + st) * 64 + c * 16 + r % 16) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                /* nibble order of k_operand: operand element i is channel i/2 + 4 (i%2) */
                const int src = BITS == 4 ? i / 2 + 4 * (i % 2) : i;
                const float x = BITS == 4 && (i / 2) % 2 ? f[src] * 0.0625f : f[src];
                o[i] = f32_to_out<true>(x);
            }
        }
    }

    static __device__ __forceinline__ void run(const KvAttnParams& p) {
        constexpr int kQBytes = kRows * kDim * 2, kMerge = kWaves * kRows * 16 * 4;
        __shared__ __attribute__((aligned(16))) char pool[kQBytes > kMerge ? kQBytes : kMerge];
        __shared__ __attribute__((aligned(16))) Scales scales[kWaves];
        __shared__ float units[kRows], qsums[kRows * kGroups];
        __shared__ float offs[kWaves][kRows], sums[kWaves][kRows];
        __shared__ float fix[kWaves][kRows][kGroups];
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;

        /* the job: heads go fastest, so that with 8 of them an XCD's L2 serves one */
        Job job;
        int i = blockIdx.x;
        const int h = i % p.heads;
        i /= p.heads;
        const int seq_rows = p.rows * p.group;
        int range, ranges;
        int64_t token0;   /* index of the slot-and-head's first token in the arrays */
        KvArrays jk, jv;
        const int prefix_jobs = p.prefix_splits * p.prefix_blocks;
        if (i < prefix_jobs) {
            range = i / p.prefix_blocks;
            ranges = p.prefix_splits;
            jk = p.prefix[0];
            jv = p.prefix[1];
            token0 = (int64_t)h * p.prefix_capacity;
            job.slot = range;
            job.row0 = (i % p.prefix_blocks) * kRows;
            job.nrows = p.batch * seq_rows - job.row0;
            job.n = job.clear = job.first = p.prefix_length;
        } else {
            i -= prefix_jobs;
            const int b = i / (p.own_splits * p.own_blocks);
            i %= p.own_splits * p.own_blocks;
            range = i / p.own_blocks;
            ranges = p.own_splits;
            jk = p.own[0];
            jv = p.own[1];
            token0 = ((int64_t)b * p.heads + h) * p.own_capacity;
            job.slot = p.prefix_splits + range;
            const int r0 = (i % p.own_blocks) * kRows;
            job.row0 = b * seq_rows + r0;
            job.nrows = seq_rows - r0;
            int n = p.lengths ? p.lengths[b] : p.max_length;
            n = n < 0 ? 0 : n > p.max_length ? p.max_length : n;
            job.n = n;
            job.first = n - p.rows;
            job.clear = job.first < 0 ? 0 : job.first;
        }
        if (job.nrows > kRows) job.nrows = kRows;
        job.k = (const char*)jk.codes + token0 * kRowBytes;
        job.v = (const char*)jv.codes + token0 * kRowBytes;
        const uint16_t* ks = lane & 16 ? jk.biases : jk.scales;
        const uint16_t* vs = lane & 16 ? jv.biases : jv.scales;
        job.scale = (lane < 32 ? ks : vs) + token0 * kGroups;
        /* ranges of whole rounds of 32 tokens a wave */
        const int rounds = (job.n + 32 * kWaves - 1) / (32 * kWaves);
        const int each = (rounds + ranges - 1) / ranges * 32 * kWaves;
        job.t0 = range * each < job.n ? range * each : job.n;
        job.t1 = job.t0 + each < job.n ? job.t0 + each : job.n;
        const int tiles = (job.nrows + 15) / 16;

        stage_queries(p, job, h, (uint16_t*)pool, units, qsums);
        __syncthreads();

        Rows st;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = rt * 16 + (lane & 15);
            st.off[rt] = kNever;
            st.sum[rt] = 0.0f;
            st.unit[rt] = units[r];
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                st.code_sum[rt][g] = st.bias_sum[rt][g] = 0.0f;
                st.qsum[rt][g] = qsums[r * kGroups + g];
            }
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) st.o[rt][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            st.mask[rt] = 0;
            if (r < job.nrows) {
                const int bm = (job.row0 + r) / p.group;
                st.mask[rt] = p.tree ? p.tree[bm] : (2u << (bm % p.rows)) - 1;
            }
        }

        int t = job.t0 + 32 * wave;
        KTile k;
        VTile v;
        float z[RT][8];
        const f16x8_t* q = (const f16x8_t*)pool;
        if (t < job.t1) {
            if (t + 32 <= job.n) load_k<false>(job, t, lane, k);
            else load_k<true>(job, t, lane, k);
        }
        while (t < job.t1) {
            const int next = t + 32 * kWaves;
            stage_scales(k.scale, lane, scales[wave]);
            if (t + 32 <= job.clear) {
                load_v<false>(job, t, lane, v);
                scores<false>(job, t, lane, tiles, k, scales[wave], q, st, z);
                if (next < job.t1) {
                    if (next + 32 <= job.n) load_k<false>(job, next, lane, k);
                    else load_k<true>(job, next, lane, k);
                }
                weigh<false>(job, t, lane, tiles, v, scales[wave], st, z);
            } else {
                load_v<true>(job, t, lane, v);
                scores<true>(job, t, lane, tiles, k, scales[wave], q, st, z);
                if (next < job.t1) load_k<true>(job, next, lane, k);
                weigh<true>(job, t, lane, tiles, v, scales[wave], st, z);
            }
            t = next;
        }

        /* the waves' rows together: offsets and sums first, then 16 columns at a time */
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = rt * 16 + (lane & 15);
            float sum = st.sum[rt];
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                float f = fmaf(-kCentre, st.code_sum[rt][g], st.bias_sum[rt][g]);
                f += __shfl_xor(f, 16);
                f += __shfl_xor(f, 32);
                if (lane < 16) fix[wave][r][g] = f;
            }
            if (lane < 16) {
                offs[wave][r] = st.off[rt];
                sums[wave][r] = sum;
            }
        }
        __syncthreads();
        const int64_t nrows = (int64_t)p.batch * seq_rows;
        const int64_t out = (job.slot * p.heads + h) * nrows + job.row0;
        if ((int)threadIdx.x < job.nrows) {
            const int r = threadIdx.x;
            float top = offs[0][r], sum = 0.0f;
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, offs[w][r]);
            for (int w = 0; w < kWaves; ++w) {
                const float f = offs[w][r] == top ? 1.0f : exp2f(offs[w][r] - top);
                sum = fmaf(sums[w][r], f, sum);
                offs[w][r] = f;   /* from here on the wave's weight */
            }
            p.part_ml[(out + r) * 2] = top;
            p.part_ml[(out + r) * 2 + 1] = sum;
        }
        float* merge = (float*)pool;
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) {
            __syncthreads();
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    merge[(wave * kRows + rt * 16 + 4 * (lane >> 4) + r) * 16 + (lane & 15)] =
                        st.o[rt][d][r];
            __syncthreads();
            const float back = odd_tile(d % kTiles) ? kUnit / 16.0f : kUnit;
            for (int e = threadIdx.x; e < job.nrows * 16; e += DFQ_KV_THREADS) {
                const int r = e / 16;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
                    sum = fmaf(fmaf(merge[w * kRows * 16 + e], back, fix[w][r][d / kTiles]),
                               offs[w][r], sum);
                p.part_o[(out + r) * kDim + d * 16 + e % 16] = sum;
            }
        }
    }
};

/* The parts of a row from all ranges, in the order of their slots: y = sum 2^(M - top) o / sum
 * 2^(M - top) l.  One workgroup a row: its waves take every fourth slot, a lane kDim / 64
 * channels. */
template <int GS, bool F16>
__device__ __forceinline__ void join(const KvAttnParams& p) {
    __shared__ float acc[kWaves][kDim], tops[kWaves], sums[kWaves];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t nrows = (int64_t)p.batch * p.rows * p.group;
    const int h = blockIdx.y, slots = p.prefix_splits + p.own_splits;
    const int64_t row = blockIdx.x, stride = nrows * p.heads, at = h * nrows + row;
    float top = kNever;
    for (int s = wave; s < slots; s += kWaves) top = fmaxf(top, p.part_ml[(s * stride + at) * 2]);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
    float sum = 0.0f, o[kDim / 64] = {};
    for (int s = wave; s < slots; s += kWaves) {
        const float off = p.part_ml[(s * stride + at) * 2], l = p.part_ml[(s * stride + at) * 2 + 1];
        const float f = off == top ? 1.0f : exp2f(off - top);
        sum = fmaf(l, f, sum);
        const float* part = p.part_o + (s * stride + at) * kDim;
#pragma unroll
        for (int i = 0; i < kDim / 64; ++i) o[i] = fmaf(part[i * 64 + lane], f, o[i]);
    }
#pragma unroll
    for (int i = 0; i < kDim / 64; ++i) acc[wave][i * 64 + lane] = o[i];
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += sums[w];
    const int64_t bm = row / p.group, q_heads = p.heads * p.group;
    const int64_t head = h * p.group + row % p.group;
    for (int d = threadIdx.x; d < kDim; d += DFQ_KV_THREADS) {
        /* channel d of group g is column (d % GS) / (GS / 16) of the group's tile d % (GS / 16) */
        constexpr int kTiles = GS / 16;
        const int e = (d / GS * kTiles + d % kTiles) * 16 + d % GS / kTiles;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v += acc[w][e];
        p.y[(bm * q_heads + head) * kDim + d] = f32_to_out<F16>(sum == 0.0f ? 0.0f : v / sum);
    }
    if (p.lse && threadIdx.x == 0)
        p.lse[bm * q_heads + head] =
            sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * 0.693147180559945309f;
}

}  // namespace

/* Built for as many row tiles as the registers hold without spilling; per_simd is the waves a
 * SIMD then has room for.  attention_tiles (verify_ops.cpp) knows which exist. */
#define DFQ_ATTN(bits, gs, name, f16, rt, per_simd)                                            \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS, per_simd) void                     \
        dfq_cache_attention_b##bits##_g##gs##_##name##_r##rt(KvAttnParams p) {                 \
        Attention<bits, gs, f16, rt>::run(p);                                                  \
    }
#define DFQ_JOIN(gs, name, f16)                                                                \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void                               \
        dfq_cache_attention_join_g##gs##_##name(KvAttnParams p) {                              \
        join<gs, f16>(p);                                                                      \
    }
#define DFQ_FORMATS(M, gs, rt, per_simd)                                  \
    M(4, gs, bf16, false, rt, per_simd) M(8, gs, bf16, false, rt, per_simd) \
    M(4, gs, f16, true, rt, per_simd) M(8, gs, f16, true, rt, per_simd)
#define DFQ_JOINS(gs) DFQ_JOIN(gs, bf16, false) DFQ_JOIN(gs, f16, true)

DFQ_JOINS(32)
DFQ_JOINS(64)
#if DFQ_HEAD_DIM == 64
DFQ_FORMATS(DFQ_ATTN, 32, 1, 3)
DFQ_FORMATS(DFQ_ATTN, 32, 2, 2)
DFQ_FORMATS(DFQ_ATTN, 32, 4, 1)
DFQ_FORMATS(DFQ_ATTN, 64, 1, 4)
DFQ_FORMATS(DFQ_ATTN, 64, 2, 3)
DFQ_FORMATS(DFQ_ATTN, 64, 4, 1)
#elif DFQ_HEAD_DIM == 128
DFQ_JOINS(128)
DFQ_FORMATS(DFQ_ATTN, 32, 1, 2)
DFQ_FORMATS(DFQ_ATTN, 32, 2, 1)
DFQ_FORMATS(DFQ_ATTN, 64, 1, 3)
DFQ_FORMATS(DFQ_ATTN, 64, 2, 2)
DFQ_FORMATS(DFQ_ATTN, 64, 4, 1)
DFQ_FORMATS(DFQ_ATTN, 128, 1, 2)
DFQ_FORMATS(DFQ_ATTN, 128, 2, 2)
DFQ_FORMATS(DFQ_ATTN, 128, 4, 1)
#elif DFQ_HEAD_DIM == 256
DFQ_JOINS(128)
DFQ_FORMATS(DFQ_ATTN, 32, 1, 1)
DFQ_FORMATS(DFQ_ATTN, 64, 1, 1)
DFQ_FORMATS(DFQ_ATTN, 128, 1, 2)
DFQ_FORMATS(DFQ_ATTN, 128, 2, 1)
#else
#error "DFQ_HEAD_DIM must be 64, 128 or 256"
#endif
