// tq_near.cuh — nearest codebook level by a shared-memory table.
#pragma once

#include "tq_common.cuh"

namespace tq {

// ── nearest level by table ─────────────────────────────────────────────────
// bin(xn) = round(16 xn + 16) is the low 6 mantissa bits of fma(xn, 16, 1.5 * 2^23 + 16)
// (one ulp is 1 at that magnitude, and round-to-nearest is monotone in xn).  Each
// boundary B_k has a bin too; for every bin j the table holds
//   cnt_j = #{k : bin(B_k) < j}   and   cand_j = the boundary with bin(B_k) = j (else +inf).
// By monotonicity every xn in bin j lies above the boundaries of lower bins and below
// those of higher bins, and no bin holds two boundaries (adjacent boundaries are at
// least 0.0945 = 1.5 bins apart), so #{k : B_k < xn} = cnt_j + [cand_j < xn]: the
// reference's nearest index for finite xn (clamping xn to [-1, 1] never changes that
// count).  |xn| <= 1 + 2^-22 keeps j in 0 .. 32 whenever 1/amax is finite; blocks with
// an infinite 1/amax (amax below 2^-128) take the compare-tree search instead.  A NaN
// xn is the canonical 0x7FFFFFFF on the GPU and falls in bin 63, whose entry gives the
// reference's NaN code (TQ3 0, TQ4 15).  Rows are replicated for the 16 lanes of a half
// warp (8-byte entries: lane l reads banks 2l and 2l + 1), so lookups never conflict.
constexpr float BIN_MAGIC = 12582928.0f;   // 1.5 * 2^23 + 16
constexpr float BIN_SCALE = 16.0f;
constexpr uint32_t BIN_MASK = 0x3Fu;
constexpr int NEAR_ROWS = 64, NEAR_REP = 16;

template <int QT>
__device__ __forceinline__ float boundary(int k) {   // B_k of src/ggml-tq.h:93-121, exact fp32
    if constexpr (QT == 2) {
        return k == 0 ? -TQ2_P0 : (k == 1 ? 0.0f : TQ2_P0);
    } else if constexpr (QT == 4) {
        constexpr float P[7] = {TQ4_P0, TQ4_P1, TQ4_P2, TQ4_P3, TQ4_P4, TQ4_P5, TQ4_P6};
        return k < 7 ? -P[6 - k] : (k == 7 ? 0.0f : P[k - 8]);
    } else {
        constexpr float P[3] = {TQ3_P0, TQ3_P1, TQ3_P2};
        return k < 3 ? -P[2 - k] : (k == 3 ? 0.0f : P[k - 4]);
    }
}

template <int QT, int THREADS = 128>
__device__ void near_table_init(uint2* __restrict__ t) {
    // one thread per row: count the boundaries of lower bins, find this bin's boundary,
    // then write the row's 16 replicas
    constexpr int NB = QT == 4 ? 15 : QT == 3 ? 7 : 3;
    for (int row = threadIdx.x; row < NEAR_ROWS; row += THREADS) {
        uint32_t cnt = QT == 4 ? 15u : 0u;   // bins past 32: only a NaN reaches them
        float cand = INFINITY;
        if (row <= 32) {
            cnt = 0;
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const float b = boundary<QT>(k);
                const int bk = (int)(__float_as_uint(__fmaf_rn(b, BIN_SCALE, BIN_MAGIC)) & BIN_MASK);
                cnt += bk < row;
                cand = bk == row ? b : cand;
            }
        }
        const uint4 e = make_uint4(__float_as_uint(cand), cnt, __float_as_uint(cand), cnt);
#pragma unroll
        for (int r = 0; r < NEAR_REP / 2; ++r) reinterpret_cast<uint4*>(t + row * NEAR_REP)[r] = e;
    }
}

// nearest indices of xn.x, xn.y; tb = shared address of the table + 8 * (lane % 16)
__device__ __forceinline__ void near_pair(float2 xn, uint32_t tb, uint32_t& i0, uint32_t& i1) {
    const float2 f = __ffma2_rn(xn, make_float2(BIN_SCALE, BIN_SCALE), make_float2(BIN_MAGIC, BIN_MAGIC));
    const uint32_t a0 = tb + ((__float_as_uint(f.x) & BIN_MASK) << 7);
    const uint32_t a1 = tb + ((__float_as_uint(f.y) & BIN_MASK) << 7);
    uint32_t c0, n0, c1, n1;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(c0), "=r"(n0) : "r"(a0));
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(c1), "=r"(n1) : "r"(a1));
    asm("{\n\t.reg .pred p;\n\tsetp.gt.f32 p, %1, %2;\n\t@p add.u32 %0, %0, 1;\n\t}" : "+r"(n0) : "f"(xn.x), "f"(__uint_as_float(c0)));
    asm("{\n\t.reg .pred p;\n\tsetp.gt.f32 p, %1, %2;\n\t@p add.u32 %0, %0, 1;\n\t}" : "+r"(n1) : "f"(xn.y), "f"(__uint_as_float(c1)));
    i0 = n0;
    i1 = n1;
}

}  // namespace tq
