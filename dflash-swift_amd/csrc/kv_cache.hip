/*
 * kv_cache.hip -- gfx950 kernels of the quantised key/value cache: rows quantised as they are
 * written, and read back.
 *
 * The format is that of the weights: per group of GS neighbouring channels of one head's row, a
 * scale s and a bias b of 16 bits and codes c of BITS bits, the value being s c + b.  A group's
 * b is its least element and s = (greatest - least) / (2^BITS - 1), each rounded once to the
 * cache's type; codes are (x - b) / s with those rounded numbers, rounded to nearest even in
 * fp32 and clamped.  A group of equal elements has s = 0 and codes 0; one whose s or b is not
 * finite (an infinite or NaN element, or a range past fp32) has s = b = NaN and codes 0, so that
 * it reads back as NaN throughout.
 *
 * Both kernels are bound by memory on long spans and by the launch on short ones.  A lane holds 8
 * channels, 16 bytes of a row, and the heads of the same rows lie side by side in the grid, so that
 * a row's bytes are touched together.  8192 rows of 8 + 8 heads of 128, 4 bits in groups of 64,
 * bf16: appended in 12.4 us (43 MB, 3.5 TB/s; 8.9 us without any arithmetic), read back in 10.2.
 * 32768 rows read in 31 us (172 MB, 5.5 TB/s; a copy of a GiB moves 5.2).  One row of 8 sequences:
 * 3.2 and 2.8 us.  The same blocks dealt out over the XCDs by heads were slower (32768 rows 37.6 us
 * for 33.9).
 */
#include "kv_params.h"
#include "qmm_device.h"

namespace {

/* 16 bytes at any 2-byte address (rows cut from a fused projection have any element offset). */
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

/* The position of row m of sequence b, or -1 where the cache has none. */
__device__ __forceinline__ int position(const int32_t* starts, int start, int b, int m,
                                        int capacity) {
    const int64_t pos = (int64_t)start + (starts ? starts[b] : 0) + m;
    return pos >= 0 && pos < capacity ? (int)pos : -1;
}

/* The code of x - bias = d, in the low bits of a float: d / s to nearest even, clamped to 0..TOP,
 * plus 1.5 2^23.  The product with a reciprocal of s is within 3 2^-24 of the quotient, relative, so
 * it rounds to the same whole number unless it lies that near to the middle of two; there the
 * division decides (one in thousands, and ties).  Dividing all of them, 8192 rows of 8 + 8 heads of
 * 128 took 16.1 us for 12.4. */
template <int TOP>
__device__ __forceinline__ uint32_t code_of(float d, float s, float inverse) {
    constexpr float kWhole = 12582912.0f, kNear = 0.5f - TOP * 4e-7f;
    const float q = __builtin_amdgcn_fmed3f(d * inverse, 0.0f, (float)TOP);
    float t = q + kWhole;
    if (fabsf(q - (t - kWhole)) > kNear)
        t = __builtin_amdgcn_fmed3f(d / s, 0.0f, (float)TOP) + kWhole;
    return __float_as_uint(t);
}

/* One group's share of a lane: 8 channels quantised and stored at token `row` of the arrays (not
 * where it is negative; every lane of a group takes part in its exchanges). */
template <int DIM, int BITS, int GS, bool F16>
__device__ __forceinline__ void append_piece(const KvArrays& o, u32x4_t raw, int lane, int64_t row) {
    constexpr int kGroups = DIM / GS;
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = elem_to_f32<F16>(raw[i] & 0xffffu);
        f[2 * i + 1] = elem_to_f32<F16>(raw[i] >> 16);
    }
    float lo = f[0], hi = f[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = fminf(lo, f[i]);
        hi = fmaxf(hi, f[i]);
    }
    /* the largest exponent: all ones in an infinity or NaN, which minima pass over */
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t most = __builtin_bit_cast(u16x2_t, raw[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i)
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, raw[i] & 0x7fff7fffu));
    const auto least_of = [](uint32_t a, uint32_t b) {
        return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b)));
    };
    const auto most_of = [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    };
    const auto larger_of = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    lo = __uint_as_float(group_of<GS / 8>(__float_as_uint(lo), least_of));
    hi = __uint_as_float(group_of<GS / 8>(__float_as_uint(hi), most_of));
    const uint32_t top = group_of<GS / 8>(most[0] > most[1] ? most[0] : most[1], larger_of);
    constexpr float kTop = (float)((1 << BITS) - 1);
    /* the least element is a number of the cache's type already */
    uint16_t s16 = F16 ? __builtin_bit_cast(uint16_t, (_Float16)((hi - lo) / kTop))
                       : __builtin_bit_cast(uint16_t, (__bf16)((hi - lo) / kTop));
    uint16_t b16 = F16 ? __builtin_bit_cast(uint16_t, (_Float16)lo)
                       : (uint16_t)(__float_as_uint(lo) >> 16);
    float s = elem_to_f32<F16>(s16);
    const float bias = elem_to_f32<F16>(b16);
    if (top >= (F16 ? 0x7c00u : 0x7f80u) || !(fabsf(s) < __builtin_inff())) {
        s16 = b16 = F16 ? 0x7e00 : 0x7fc0;
        s = 0.0f;
    }
    /* no scale, no codes: the products are then 0; a denormal scale's reciprocal may not be finite,
     * and the quotients are divided from its largest power of two */
    float up = 1.0f;
    if (s < 1.1754944e-38f) up = 0x1p40f;
    const float by = s * up, inverse = s > 0.0f ? __builtin_amdgcn_rcpf(by) : 0.0f;
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = code_of<(1 << BITS) - 1>((f[i] - bias) * up, by, inverse);
    if (row < 0) return;
    uint32_t* w = o.codes + row * (DIM * BITS / 32) + lane * (BITS / 4);
    /* the codes above each other; what 1.5 2^23 adds to the sums is the same for all */
    constexpr int kPer = 32 / BITS;
    constexpr uint32_t kExtra = BITS == 4 ? 0x4b400000u * 0x11111111u : 0x4b400000u * 0x01010101u;
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
        uint32_t v = c[kPer * i + kPer - 1];
#pragma unroll
        for (int j = kPer - 2; j >= 0; --j) v = (v << BITS) + c[kPer * i + j];
        w[i] = v - kExtra;
    }
    if (lane % (GS / 8) == 0) {
        o.scales[row * kGroups + lane / (GS / 8)] = s16;
        o.biases[row * kGroups + lane / (GS / 8)] = b16;
    }
}

/* One workgroup: DFQ_KV_THREADS * 8 / DIM tokens of one head of one sequence; a lane holds 8
 * channels of K and of V, so that a group is GS / 8 neighbouring lanes. */
template <int DIM, int BITS, int GS, bool F16>
__device__ __forceinline__ void append_rows(const KvAppendParams& p) {
    constexpr int kLanes = DIM / 8, kTokens = DFQ_KV_THREADS / kLanes;
    const int b = blockIdx.z, lane = threadIdx.x % kLanes;
    const int h = blockIdx.x % p.heads;
    const int64_t m = (int64_t)(blockIdx.x / p.heads) * kTokens + threadIdx.x / kLanes;
    /* rows past the end follow row 0 through the exchanges and store nothing */
    const int64_t mm = m < p.rows ? m : 0;
    const int64_t at = ((int64_t)b * p.rows + mm) * p.row_stride + h * DIM + lane * 8;
    const u32x4_t k = *(const u32x4_any*)(p.in[0] + at), v = *(const u32x4_any*)(p.in[1] + at);
    const int pos = m < p.rows ? position(p.starts, p.start, b, (int)m, p.capacity) : -1;
    const int64_t row = pos < 0 ? -1 : ((int64_t)b * p.heads + h) * p.capacity + pos;
    append_piece<DIM, BITS, GS, F16>(p.out[0], k, lane, row);
    append_piece<DIM, BITS, GS, F16>(p.out[1], v, lane, row);
}

/* The same split, K or V: a lane's 8 channels of one token back as values in the cache's type or
 * (out_dt 2) fp32, each rounded once.  Positions that the cache does not have read as zero. */
template <int DIM, int BITS, int GS, bool F16>
__device__ __forceinline__ void read_rows(const KvReadParams& p, int out_dt) {
    constexpr int kLanes = DIM / 8, kTokens = DFQ_KV_THREADS / kLanes, kGroups = DIM / GS;
    const int kv = blockIdx.z & 1, b = blockIdx.z >> 1, lane = threadIdx.x % kLanes;
    const int h = blockIdx.x % p.heads;
    const int64_t m = (int64_t)(blockIdx.x / p.heads) * kTokens + threadIdx.x / kLanes;
    if (m >= p.rows || !p.out[kv]) return;
    const int pos = position(p.starts, p.start, b, (int)m, p.capacity);
    float f[8] = {};
    if (pos >= 0) {
        const KvArrays& a = p.in[kv];
        const int64_t row = ((int64_t)b * p.heads + h) * p.capacity + pos;
        const uint32_t* w = a.codes + row * (DIM * BITS / 32) + lane * (BITS / 4);
        const float s = elem_to_f32<F16>(a.scales[row * kGroups + lane / (GS / 8)]);
        const float bias = elem_to_f32<F16>(a.biases[row * kGroups + lane / (GS / 8)]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t c = BITS == 4 ? w[0] >> (4 * i) & 15u : w[i / 4] >> (8 * (i % 4)) & 255u;
            f[i] = fmaf(s, (float)c, bias);
        }
    }
    const int64_t at = (((int64_t)b * p.rows + m) * p.heads + h) * DIM + lane * 8;
    if (out_dt == 2) {
        float* o = (float*)p.out[kv] + at;
#pragma unroll
        for (int i = 0; i < 8; i += 4)
            __builtin_nontemporal_store(f32x4_t{f[i], f[i + 1], f[i + 2], f[i + 3]},
                                        (f32x4_t*)(o + i));
        return;
    }
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = F16 ? f32_to_out<true>(f[2 * i]) | (uint32_t)f32_to_out<true>(f[2 * i + 1]) << 16
                   : f32_to_out<false>(f[2 * i]) | (uint32_t)f32_to_out<false>(f[2 * i + 1]) << 16;
    /* written once and not read here: past the caches (32768 tokens, 172 MB, 43 -> 34 us) */
    __builtin_nontemporal_store(v, (u32x4_t*)((uint16_t*)p.out[kv] + at));
}

}  // namespace

#define DFQ_KV_KERNELS(dim, bits, gs, name, f16)                                               \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void                               \
        dfq_cache_append_d##dim##_b##bits##_g##gs##_##name(KvAppendParams p) {                 \
        append_rows<dim, bits, gs, f16>(p);                                                    \
    }                                                                                          \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void                               \
        dfq_cache_read_d##dim##_b##bits##_g##gs##_##name(KvReadParams p, int out_dt) {         \
        read_rows<dim, bits, gs, f16>(p, out_dt);                                              \
    }
#define DFQ_KV_DTYPES(dim, bits, gs)            \
    DFQ_KV_KERNELS(dim, bits, gs, bf16, false)  \
    DFQ_KV_KERNELS(dim, bits, gs, f16, true)
#define DFQ_KV_BITS(dim, gs) DFQ_KV_DTYPES(dim, 4, gs) DFQ_KV_DTYPES(dim, 8, gs)
DFQ_KV_BITS(64, 32)
DFQ_KV_BITS(64, 64)
DFQ_KV_BITS(128, 32)
DFQ_KV_BITS(128, 64)
DFQ_KV_BITS(128, 128)
DFQ_KV_BITS(256, 32)
DFQ_KV_BITS(256, 64)
DFQ_KV_BITS(256, 128)
