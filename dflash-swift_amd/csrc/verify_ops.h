/*
 * verify_ops.h -- what the host sources of a verify pass's operators share: embedding and loading of
 * their kernels, and small helpers.
 */
#ifndef DFQ_VERIFY_OPS_H
#define DFQ_VERIFY_OPS_H

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>
#include <new>

#include "kv_params.h"
#include "qmm_internal.h"

/* A gfx950 code object embedded under a name. */
#define DFQ_EMBED(name, path)                      \
    __asm__(".section .rodata.dfq_verify_hsaco,\"a\",@progbits\n" \
            ".p2align 12\n"                        \
            ".globl " #name "\n"                   \
            ".hidden " #name "\n"                  \
            #name ":\n"                            \
            ".incbin \"" path "\"\n"              \
            ".byte 0\n"                            \
            ".previous\n");                        \
    extern "C" const char name[];

namespace dfq {

inline dfq_status hip_error(hipError_t e, const char* what) {
    return fail(DFQ_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

/* A context's kernels of one group: Ops is a LoadedOps with its kGroup and resolve(). */
template <typename Ops>
dfq_status load_ops(LoadedOps** out) {
    Ops* o = new (std::nothrow) Ops();
    if (!o) return fail(DFQ_ERR_HIP, "out of host memory");
    const dfq_status s = o->resolve();
    if (s) {
        delete o;
        return s;
    }
    *out = o;
    return DFQ_OK;
}
template <typename Ops>
dfq_status ops_of(dfq_ctx* ctx, const Ops** out) {
    const LoadedOps* o;
    const dfq_status s = ctx_ops(ctx, Ops::kGroup, load_ops<Ops>, &o);
    if (s == DFQ_OK) *out = static_cast<const Ops*>(o);
    return s;
}

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

inline size_t dtype_size(dfq_dtype t) { return t == DFQ_F32 ? 4 : 2; }

/* The launch grid's limits in y and z, and of x in workgroups of DFQ_KV_THREADS: a grid has fewer
 * than 2^32 threads along it. */
constexpr int kMostGrid = 65535;
constexpr int64_t kMostGroups = ((int64_t)1 << 32) / DFQ_KV_THREADS - 1;

/* by 0: of a part of the call that is not there, and nothing is divided */
inline Divisor divisor(int by) {
    const uint64_t d = by > 0 ? by : 1;
    int shift = 0;
    while ((1ull << shift) < d) ++shift;
    return {(uint32_t)by, (uint32_t)((((1ull << shift) - d) << 32) / d + 1), shift};
}

}  // namespace dfq

#endif
