/*
 * verify_ops.h -- what the host sources of a verify pass's operators share: their kernels, loaded
 * together with a context's first call of one of them, and small helpers.
 */
#ifndef DFQ_VERIFY_OPS_H
#define DFQ_VERIFY_OPS_H

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "kv_params.h"
#include "qmm_internal.h"

namespace dfq {

/* One format of a cache: [head_dim 64/128/256][bits 4/8][group 32/64/128][bf16/f16]; groups wider
 * than the head have no kernels. */
struct CacheKernels {
    hipFunction_t append = nullptr, read = nullptr, join = nullptr;
    hipFunction_t attention[2] = {};  // up to 1 and 2 row tiles (see attention_tiles)
    int resident[2] = {};             // their workgroups that a CU holds at once
};

struct AcceptKernels {
    hipFunction_t sums[2] = {}, weigh[2] = {}, rest = nullptr;   // [sums in fp32/64 bits]
};

struct VerifyOps {
    hipModule_t kv = nullptr, logprobs = nullptr, attention[3] = {}, rope = nullptr,
                sample = nullptr;
    CacheKernels cache[3][2][3][2];
    hipFunction_t logprobs_part[3] = {}, logprobs_join[3] = {};  // [bf16/f16/f32]
    hipFunction_t rotate[2][3][3] = {};  // [alone/with norms][halves/pairs/any][bf16/f16/f32]
    AcceptKernels accept[3];             // [bf16/f16/f32]
};

inline dfq_status hip_error(hipError_t e, const char* what) {
    return fail(DFQ_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

inline size_t dtype_size(dfq_dtype t) { return t == DFQ_F32 ? 4 : 2; }

/* The launch grid's limits in y and z. */
constexpr int kMostGrid = 65535;

/* by 0: of a part of the call that is not there, and nothing is divided */
inline Divisor divisor(int by) {
    const uint64_t d = by > 0 ? by : 1;
    int shift = 0;
    while ((1ull << shift) < d) ++shift;
    return {(uint32_t)by, (uint32_t)((((1ull << shift) - d) << 32) / d + 1), shift};
}

}  // namespace dfq

#endif
