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

/* Minimum or maximum over the L lanes (a power of two, up to 16) of a group. */
template <int L, bool MAX>
__device__ __forceinline__ float group_best(float v) {
#pragma unroll
    for (int d = 1; d < L; d *= 2) {
        const float o = __shfl_xor(v, d);
        v = MAX ? fmaxf(v, o) : fminf(v, o);
    }
    return v;
}

/* One workgroup: DFQ_KV_THREADS * 8 / DIM tokens of one head of one sequence, K or V; a lane
 * holds 8 channels, so that a group is GS / 8 neighbouring lanes. */
template <int DIM, int BITS, int GS, bool F16>
__device__ __forceinline__ void append_rows(const KvAppendParams& p) {
    constexpr int kLanes = DIM / 8, kTokens = DFQ_KV_THREADS / kLanes, kGroups = DIM / GS;
    const int lane = threadIdx.x % kLanes, m = blockIdx.x * kTokens + threadIdx.x / kLanes;
    const int h = blockIdx.y, kv = blockIdx.z & 1, b = blockIdx.z >> 1;
    /* rows past the end follow row 0 through the exchanges and store nothing */
    const int mm = m < p.rows ? m : 0;
    const uint16_t* x = p.in[kv] + ((int64_t)b * p.rows + mm) * p.row_stride + h * DIM + lane * 8;
    const u32x4_any raw = *(const u32x4_any*)x;
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = elem_to_f32<F16>(raw[i] & 0xffffu);
        f[2 * i + 1] = elem_to_f32<F16>(raw[i] >> 16);
    }
    float lo = f[0], hi = f[0], odd = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, f[i]);
        hi = fmaxf(hi, f[i]);
        odd = fmaxf(odd, f[i] != f[i] ? 1.0f : 0.0f); /* the minimum passes NaN over */
    }
    lo = group_best<GS / 8, false>(lo);
    hi = group_best<GS / 8, true>(hi);
    odd = group_best<GS / 8, true>(odd);
    constexpr float kTop = (float)((1 << BITS) - 1);
    uint16_t s16 = f32_to_out<F16>((hi - lo) / kTop), b16 = f32_to_out<F16>(lo);
    float s = elem_to_f32<F16>(s16);
    const float bias = elem_to_f32<F16>(b16);
    if (odd != 0.0f || !(fabsf(s) < __builtin_inff()) || !(fabsf(bias) < __builtin_inff())) {
        s16 = b16 = F16 ? 0x7e00 : 0x7fc0;
        s = 0.0f;
    }
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = s > 0.0f ? rintf((f[i] - bias) / s) : 0.0f;
        c[i] = (uint32_t)fminf(fmaxf(v, 0.0f), kTop);
    }
    const int pos = m < p.rows ? position(p.starts, p.start, b, m, p.capacity) : -1;
    if (pos < 0) return;
    const KvArrays& o = p.out[kv];
    const int64_t row = ((int64_t)b * p.heads + h) * p.capacity + pos;
    uint32_t* w = o.codes + row * (DIM * BITS / 32) + lane * (BITS / 4);
    if constexpr (BITS == 4) {
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) v |= c[i] << (4 * i);
        w[0] = v;
    } else {
        w[0] = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        w[1] = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
    }
    if (lane % (GS / 8) == 0) {
        o.scales[row * kGroups + lane / (GS / 8)] = s16;
        o.biases[row * kGroups + lane / (GS / 8)] = b16;
    }
}

/* The same split: a lane's 8 channels of one token back as OUT values (0 bf16, 1 fp16, 2 fp32),
 * each rounded once.  Positions that the cache does not have read as zero. */
template <int DIM, int BITS, int GS, bool F16>
__device__ __forceinline__ void read_rows(const KvReadParams& p, int out_dt) {
    constexpr int kLanes = DIM / 8, kTokens = DFQ_KV_THREADS / kLanes, kGroups = DIM / GS;
    const int lane = threadIdx.x % kLanes, m = blockIdx.x * kTokens + threadIdx.x / kLanes;
    const int h = blockIdx.y, kv = blockIdx.z & 1, b = blockIdx.z >> 1;
    if (m >= p.rows || !p.out[kv]) return;
    const int pos = position(p.starts, p.start, b, m, p.capacity);
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
        for (int i = 0; i < 8; ++i) o[i] = f[i];
        return;
    }
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = out_dt == 1 ? f32_to_out<true>(f[2 * i]) | (uint32_t)f32_to_out<true>(f[2 * i + 1]) << 16
                           : f32_to_out<false>(f[2 * i]) | (uint32_t)f32_to_out<false>(f[2 * i + 1]) << 16;
    *(u32x4_t*)((uint16_t*)p.out[kv] + at) = v;
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
