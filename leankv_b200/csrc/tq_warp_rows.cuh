// tq_warp_rows.cuh — head rows held by a whole warp, D / 32 consecutive elements to a lane.
#pragma once

#include "tq_common.cuh"

namespace tq {

// E consecutive elements (4 or 8) as float32
template <int E> __device__ __forceinline__ void load_some(int dtype, const void* p, int64_t at, float (&v)[E]) {
    if (dtype == DT_F32) {
#pragma unroll
        for (int j = 0; j < E / 4; ++j) {
            const float4 x = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at)[j];
            v[4 * j] = x.x; v[4 * j + 1] = x.y; v[4 * j + 2] = x.z; v[4 * j + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < E / 4; ++j) {
            const uint2 x = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at)[j];
            const uint32_t w[4] = {x.x & 0xFFFFu, x.x >> 16, x.y & 0xFFFFu, x.y >> 16};
#pragma unroll
            for (int k = 0; k < 4; ++k) v[4 * j + k] = dtype == DT_F16 ? f16_bits_to_float(w[k]) : bf16_bits_to_float(w[k]);
        }
    }
}
// Hadamard transform of a row held E elements to a lane of the warp
template <int E> __device__ __forceinline__ void fwht_warp(float (&v)[E], float norm) {
#pragma unroll
    for (int h = 1; h < E; h *= 2)
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (j & h) continue;
            const float a = v[j], b = v[j + h];
            v[j] = a + b;
            v[j + h] = a - b;
        }
#pragma unroll
    for (int bit = 1; bit < 32; bit *= 2) {
        const float sg = (threadIdx.x & bit) ? -1.0f : 1.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = fmaf(v[j], sg, __shfl_xor_sync(0xffffffffu, v[j], bit));
    }
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] *= norm;
}
}  // namespace tq
