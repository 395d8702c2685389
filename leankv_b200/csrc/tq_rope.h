// tq_rope.h — internal interface of the rotary and rotary-append kernels.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace tq {

constexpr int Q8_BLOCK = 16;   // token slots that share one scale of an 8-bit page

// Rotation of head rows by position.  Pair i of a row turns by the angle p * inv_freq[i], p the token's
// position on axis axis[i] (axis null: axis 0).  positions [n_axes][batch][n_new], or null: the token's
// slot (first[b] + t; first null: t).
struct Rope {
    const double* inv_freq = nullptr;   // device [rotary_dim / 2]; null: no rotation
    const int32_t* axis = nullptr;      // device [rotary_dim / 2]
    const int32_t* positions = nullptr;
    int n_axes = 1, rotary_dim = 0;
    int interleaved = 0;                // pairs (2i, 2i + 1) instead of (i, i + rotary_dim / 2)
    int inverse = 0;
    double scale = 1.0;
};

// rows [batch][heads][n_new][head_dim] at element strides; the last dimension is contiguous
struct HeadRows {
    const void* src = nullptr;
    void* dst = nullptr;
    int heads = 0;
    int64_t ss[3] = {0, 0, 0};   // batch, head, token
    int64_t ds[3] = {0, 0, 0};
};

struct RotaryRun {
    int batch = 0, head_dim = 0, dtype = 0;
    int64_t n_new = 0;
    HeadRows x[2];
    Rope rope;
};

struct PoolDst {
    uint8_t* pool = nullptr;
    float* scale = nullptr;   // Q8: [num_pages][n_kv_heads][page_size / Q8_BLOCK]
    int type = 4;
};

struct RotaryAppendRun {
    int batch = 0, head_dim = 0, n_kv_heads = 0, dtype = 0;
    int64_t n_new = 0;
    HeadRows k, v, q;         // k, v: src only; q.heads == 0: no queries
    Rope rope;
    PoolDst kd, vd;
    const int32_t* pages = nullptr;
    int64_t max_pages = 0, num_pages = 0;
    int page_shift = 4;
    const int32_t* pos = nullptr;       // first slot of each sequence, null: 0
    const int32_t* new_len = nullptr;   // rows of each sequence that are stored, null: n_new
    int rotate = 1;
    float norm = 1.0f;
    int32_t* overflow = nullptr;
};

cudaError_t launch_rotary(const RotaryRun& r, cudaStream_t st);
cudaError_t launch_rotary_append(const RotaryAppendRun& r, cudaStream_t st);
cudaError_t launch_dequantize_q8(const int8_t* code, const float* scale, void* y, int out_dtype, int64_t n_blocks,
                                 int head_dim, cudaStream_t st);

}  // namespace tq
