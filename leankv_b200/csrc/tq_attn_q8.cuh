// tq_attn_q8.cuh — device helpers shared by the attention kernels over 8-bit pages.
#pragma once

#include "tq_attn_q8.h"
#include "tq_rows.cuh"

namespace tq {

// weights are 2^(s + log2 vs - m + Q8_SHIFT); a row's m moves when a score exceeds it by more than Q8_SLACK
constexpr float Q8_SHIFT = 6.0f, Q8_SLACK = 8.0f;
// What stands in for the scale of a block of zero values, whose weights still count: 1 / vs times weights of up to
// 2^(Q8_SHIFT + Q8_SLACK) is summed in fp32, so 2^26 tokens of such blocks stay below 2^128 (with 2^-100 it was 2^14
// tokens: a head of zero values behind 131072 tokens could give NaN).  Not larger: a block of zero values that has
// nearly all of a row's weight lifts the row's maximum, and the other blocks' weights with it towards f16's end.
constexpr float Q8_ZERO_SCALE = 0x1p-88f;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void load16(const void* p, int64_t at, float (&v)[16]) {
    float a[8], b[8];
    load8<T>(static_cast<const T*>(p) + at, a);
    load8<T>(static_cast<const T*>(p) + at + 8, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) { v[j] = a[j]; v[8 + j] = b[j]; }
}
__device__ __forceinline__ void load_row16(int dtype, const void* p, int64_t at, float (&v)[16]) {
    if (dtype == DT_F32) load16<float>(p, at, v);
    else if (dtype == DT_F16) load16<__half>(p, at, v);
    else load16<__nv_bfloat16>(p, at, v);
}
template <typename T>
__device__ __forceinline__ void put16(void* p, int64_t at, const float (&v)[16]) {
    float a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { a[j] = v[j]; b[j] = v[8 + j]; }
    store8<T>(static_cast<T*>(p) + at, a);
    store8<T>(static_cast<T*>(p) + at + 8, b);
}
__device__ __forceinline__ void store_row16(int dtype, void* p, int64_t at, const float (&v)[16]) {
    if (dtype == DT_F32) put16<float>(p, at, v);
    else if (dtype == DT_F16) put16<__half>(p, at, v);
    else put16<__nv_bfloat16>(p, at, v);
}

struct SeqLens {
    int len, q_len;   // cached tokens (this step's included), query tokens
};
__device__ __forceinline__ SeqLens seq_lens(const Q8Run& r, int b) {
    const int64_t cap = r.max_pages << r.page_shift;
    int64_t len = r.kv_len[b], ql = r.q_len ? r.q_len[b] : r.n;
    len = len < 0 ? 0 : (len > cap ? cap : len);
    ql = ql < 0 ? 0 : (ql > r.n ? r.n : ql);
    return {(int)len, (int)ql};
}
// last token that query token i sees (-1: none)
__device__ __forceinline__ int last_seen(const Q8Run& r, const SeqLens& s, int i) {
    if (i >= s.q_len) return -1;
    const int lim = r.causal ? s.len - s.q_len + i : s.len - 1;
    return lim < 0 ? -1 : lim;
}

// Trees of drafted nodes.  Node i of a sequence is its cached token len - q_len + i; it sees all tokens before the
// nodes and those nodes that its mask has.  last_before: the last token that it sees whatever the mask says, -1 if there
// is none, -2 for a row that sees nothing (padding, nodes before the cache's first token).
__device__ __forceinline__ int last_before(const SeqLens& s, int i) {
    const int base = s.len - s.q_len;
    if (i >= s.q_len || base + i < 0) return -2;
    return base > 0 ? base - 1 : -1;
}
__device__ __forceinline__ const uint32_t* node_mask(const Q8Run& r, int b, int i) {
    return r.tree + b * r.tree_stride + (int64_t)i * r.tree_words;
}
// bits of the nodes node0 .. node0 + 15 (node0 of any sign), those of 0 .. nodes - 1 only; a row without nodes has no mask
__device__ __forceinline__ uint32_t mask16(const uint32_t* mask, int words, int node0, int nodes) {
    if (nodes <= 0 || node0 <= -16 || node0 >= nodes) return 0;
    const int w = node0 >> 5;
    const uint32_t lo = w >= 0 ? mask[w] : 0u, hi = w + 1 < words ? mask[w + 1] : 0u;
    uint32_t bits = __funnelshift_r(lo, hi, node0 & 31) & 0xFFFFu;
    if (nodes - node0 < 16) bits &= (1u << (nodes - node0)) - 1u;
    return bits;
}

// the 16-token block of a (sequence, KV head): its index in the pool (codes at 16 D times it, scale at it), or
// -1 for a page outside the pool
__device__ __forceinline__ int block_at(const Q8Run& r, int b, int h, int block) {
    const int per = r.page_shift - 4;   // log2 blocks per page
    const int32_t pg = r.pages[(int64_t)b * r.max_pages + (block >> per)];
    if (pg < 0 || pg >= r.num_pages) return -1;
    return (int)((((int64_t)pg * r.Hkv + h) << per) + (block & ((1 << per) - 1)));
}

}  // namespace tq
