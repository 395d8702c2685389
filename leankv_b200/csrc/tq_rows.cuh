// tq_rows.cuh — head rows in registers: 8-element vector loads and stores, and the Hadamard transform of rows
// held 16 elements to a lane.
#pragma once

#include "tq_common.cuh"

namespace tq {

// 8 elements as loaded
template <typename T> struct Raw8 { uint4 w[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void store_raw8(T* p, const Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&v)[8]) {
    v[0] = __uint_as_float(r.w[0].x); v[1] = __uint_as_float(r.w[0].y); v[2] = __uint_as_float(r.w[0].z); v[3] = __uint_as_float(r.w[0].w);
    v[4] = __uint_as_float(r.w[1].x); v[5] = __uint_as_float(r.w[1].y); v[6] = __uint_as_float(r.w[1].z); v[7] = __uint_as_float(r.w[1].w);
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float (&v)[8]) {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void unpack8(const Raw8<__half>& r, float (&v)[8]) {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) { unpack8(load_raw8<T>(p), v); }
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]);
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
template <> __device__ __forceinline__ void store8<__half>(__half* p, const float (&v)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

// Hadamard stages of a row of D elements held 16 to a lane by D / 16 consecutive lanes, in the reference's
// order (h = 1, 2, 4, ...), each a correctly rounded sum and difference, then the factor 1 / sqrt(D).
template <int D>
__device__ __forceinline__ void fwht16(float (&v)[16], float norm) {
    const float2 m1 = make_float2(-1.0f, -1.0f);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        const float a = v[j], b = v[j + 1];
        v[j] = __fadd_rn(a, b);
        v[j + 1] = __fsub_rn(a, b);
    }
#pragma unroll
    for (int h = 2; h < 16; h *= 2) {
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            if (j & h) continue;
            const float2 a = make_float2(v[j], v[j + 1]), b = make_float2(v[j + h], v[j + h + 1]);
            const float2 s = __fadd2_rn(a, b), d = __ffma2_rn(b, m1, a);
            v[j] = s.x; v[j + 1] = s.y; v[j + h] = d.x; v[j + h + 1] = d.y;
        }
    }
#pragma unroll
    for (int bit = 1; bit < D / 16; bit *= 2) {
        const float sg = (threadIdx.x & bit) ? -1.0f : 1.0f;   // lower: self + other, upper: other - self
        const float2 sg2 = make_float2(sg, sg);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float p0 = __shfl_xor_sync(0xffffffffu, v[j], bit), p1 = __shfl_xor_sync(0xffffffffu, v[j + 1], bit);
            const float2 s = __ffma2_rn(make_float2(v[j], v[j + 1]), sg2, make_float2(p0, p1));
            v[j] = s.x; v[j + 1] = s.y;
        }
    }
    const float2 n2 = make_float2(norm, norm);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        const float2 s = __fmul2_rn(make_float2(v[j], v[j + 1]), n2);
        v[j] = s.x; v[j + 1] = s.y;
    }
}

}  // namespace tq
