/*
 * logprobs.hip -- gfx950 kernels of the log probabilities of given tokens, with the entropy and
 * the top alternatives of each row of logits.
 *
 * With m the largest logit of a row and l = sum e^(x - m): the log probability of token t is
 * x_t - m - log l, the entropy log l - sum (x - m) e^(x - m) / l, in fp32.  A token of
 * probability 0 (a logit of -inf) adds nothing to the entropy.  Alternatives are ordered by
 * logit, ties to the lowest index, NaN left out.
 */
#include "kv_params.h"
#include "qmm_device.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

/* Order of a logit: larger first, then the lower index; NaN below every number (0). */
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (uint64_t)(u >> 31 ? ~u : u | 0x80000000u) << 32 | (uint32_t)~i;
}

__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u);
}

template <int DT>
__device__ __forceinline__ void logprobs_row(const LogprobParams& p) {
    __shared__ float red[3][DFQ_KV_THREADS / 64];
    __shared__ uint64_t keys[DFQ_KV_THREADS / 64];
    const int tid = threadIdx.x, r = blockIdx.x;
    const char* row = (const char*)p.logits + (int64_t)r * p.row_stride * (DT == 2 ? 4 : 2);
    float m = -__FLT_MAX__;
    for (int i = tid; i < p.vocab; i += DFQ_KV_THREADS) m = fmaxf(m, load_any(row, DT, i));
    for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    if (tid % 64 == 0) red[0][tid / 64] = m;
    __syncthreads();
    for (int w = 0; w < DFQ_KV_THREADS / 64; ++w) m = fmaxf(m, red[0][w]);
    float l = 0.0f, e = 0.0f;
    for (int i = tid; i < p.vocab; i += DFQ_KV_THREADS) {
        const float x = load_any(row, DT, i) - m, w = exp2f(x * kLog2e);
        l += w;
        e = fmaf(fmaxf(x, -1000.0f), w, e);
    }
    for (int d = 1; d < 64; d *= 2) {
        l += __shfl_xor(l, d);
        e += __shfl_xor(e, d);
    }
    if (tid % 64 == 0) {
        red[1][tid / 64] = l;
        red[2][tid / 64] = e;
    }
    __syncthreads();
    l = e = 0.0f;
    for (int w = 0; w < DFQ_KV_THREADS / 64; ++w) {
        l += red[1][w];
        e += red[2][w];
    }
    /* no number above -inf: no distribution */
    const float log_l = l > 0.0f ? logf(l) : __builtin_nanf("");
    if (tid == 0) {
        if (p.entropy) p.entropy[r] = log_l - e / l;
        if (p.tokens) {
            const int t = p.tokens[r];
            p.logprobs[r] = t >= 0 && t < p.vocab ? load_any(row, DT, t) - m - log_l
                                                  : __builtin_nanf("");
        }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        uint64_t best = 0;
        for (int i = tid; i < p.vocab; i += DFQ_KV_THREADS) {
            const uint64_t key = order_key(load_any(row, DT, i), (uint32_t)i);
            if (key < last && key > best) best = key;
        }
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_xor((unsigned long long)best, d);
            best = o > best ? o : best;
        }
        __syncthreads();
        if (tid % 64 == 0) keys[tid / 64] = best;
        __syncthreads();
        for (int w = 0; w < DFQ_KV_THREADS / 64; ++w) best = keys[w] > best ? keys[w] : best;
        last = best;
        if (tid == 0) {
            p.top_tokens[(int64_t)r * p.top + k] = best ? (int32_t)~(uint32_t)best : -1;
            p.top_logprobs[(int64_t)r * p.top + k] =
                best ? key_value(best) - m - log_l : __builtin_nanf("");
        }
    }
}

}  // namespace

#define DFQ_LOGPROB_KERNEL(name, dt)                                             \
    extern "C" __global__ __launch_bounds__(DFQ_KV_THREADS) void                 \
        dfq_token_logprobs_##name(LogprobParams p) {                             \
        logprobs_row<dt>(p);                                                     \
    }
DFQ_LOGPROB_KERNEL(bf16, 0)
DFQ_LOGPROB_KERNEL(f16, 1)
DFQ_LOGPROB_KERNEL(f32, 2)
