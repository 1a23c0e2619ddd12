/*
 * logit_piece.h -- 16 bytes of a row of logits (bf16, fp16 or fp32, any element alignment), the
 * part that a lane takes at once.
 */
#ifndef DFQ_LOGIT_PIECE_H
#define DFQ_LOGIT_PIECE_H

#include "kv_device.h"

namespace {

template <int DT>
struct LogitPiece {
    static constexpr int kN = DT == 2 ? 4 : 8;       /* logits of 16 bytes              */

    /* Logits i .. of a row; those from `end` on are -inf and are not read. */
    static __device__ __forceinline__ u32x4_t load(const char* row, int i, int end) {
        constexpr int kSize = 16 / kN;
        if (i + kN <= end) return *(const u32x4_any*)(row + (int64_t)i * kSize);
        u32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == 2) {
                v[j] = i + j < end ? *(const uint32_t*)(row + (int64_t)(i + j) * 4) : 0xff800000u;
            } else {
                constexpr uint32_t kInf = DT == 1 ? 0xfc00u : 0xff80u;
                const uint16_t* p = (const uint16_t*)row + i + 2 * j;
                v[j] = (i + 2 * j < end ? p[0] : kInf) | (i + 2 * j + 1 < end ? p[1] : kInf) << 16;
            }
        }
        return v;
    }

    static __device__ __forceinline__ void widen(u32x4_t v, float (&x)[kN]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == 2) {
                x[j] = __uint_as_float(v[j]);
            } else {
                x[2 * j] = elem_to_f32<DT == 1>(v[j] & 0xffffu);
                x[2 * j + 1] = elem_to_f32<DT == 1>(v[j] >> 16);
            }
        }
    }

    static __device__ __forceinline__ float largest(const float (&x)[kN]) {
        float m = x[0];
#pragma unroll
        for (int j = 1; j < kN; ++j) m = fmaxf(m, x[j]);
        return m;
    }
};

}  // namespace

#endif
