/*
 * kv_device.h -- device helpers shared by the rotation, sampled-accept and log-probability kernels.
 */
#ifndef DFQ_KV_DEVICE_H
#define DFQ_KV_DEVICE_H

#include "kv_params.h"
#include "qmm_device.h"

namespace {

/* 16 bytes at any element's address. */
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

/* n / by.  (The attention's 32-bit sum, in its own file, took one block's head norms here from 4.56 to
 * 4.62 us.) */
__device__ __forceinline__ int divided(int n, const Divisor& d) {
    return (int)((n + (uint64_t)((uint64_t)(uint32_t)n * d.mul >> 32)) >> d.shift);
}

}  // namespace

#endif
