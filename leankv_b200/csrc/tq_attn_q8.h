// tq_attn_q8.h — internal interface of the attention kernels over 8-bit pages.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace tq {

struct Q8Run {
    int B = 0, Hq = 0, Hkv = 0, grp = 1, D = 0;
    int64_t n = 0;                 // query tokens of each sequence (padded)
    const void* q = nullptr;
    int q_dtype = 0;
    int64_t qs[3] = {0, 0, 0};     // element strides: batch, head, token
    void* out = nullptr;
    int out_dtype = 0;
    int64_t os[3] = {0, 0, 0};
    const int8_t* k = nullptr;     // [num_pages][Hkv][page][D]
    const int8_t* v = nullptr;
    const float* ks = nullptr;     // [num_pages][Hkv][page / 16]
    const float* vs = nullptr;
    const int32_t* pages = nullptr;
    int64_t max_pages = 0, num_pages = 0;
    int page_shift = 4;
    const int32_t* kv_len = nullptr;
    const int32_t* q_len = nullptr;   // null: n
    int max_len = 0;                  // the caller's bound of kv_len
    float sm_scale = 0.0f;
    int causal = 1, rotate_q = 1, v_rotated = 1;
    float norm = 1.0f;             // 1 / sqrt(D) of the Hadamard transform
    float* lse = nullptr;          // [B][Hq][n]
    int32_t* status = nullptr;
};

// Work split: a unit is one (sequence, KV head, tile of rows); `splits` CTAs share its tokens.
struct Q8Plan {
    int rows = 16;                 // query rows per unit
    int row_tiles = 1;             // units per (sequence, KV head)
    int splits = 1;
    bool lo = false;               // q' as two f16 terms
    bool prompt = false;           // the tcgen05 kernel:
    bool direct = false;           // which converts codes itself, or reads tiles from the work memory:
    int tiles_max = 0;             // tiles of a pair's tokens
    int pairs_pass = 0;            // (sequence, KV head) pairs that run at a time: all, or as many as have tiles in the work memory
    size_t tile_bytes = 0;
};

Q8Plan q8_plan(int B, int Hkv, int grp, int D, int64_t n, int64_t max_len, bool lo);
size_t q8_workspace_bytes(int D, const Q8Plan& p);
int q8_prompt_rows(int64_t pairs, int64_t rows, int D, bool direct, bool lo);
void q8_prompt_tiles(int64_t pairs, int D, int64_t max_len, Q8Plan* p);
cudaError_t launch_attention_q8_prompt(const Q8Run& r, const Q8Plan& p, float* part, float* part_lse, void* tiles, cudaStream_t st);
cudaError_t q8_default_status(int32_t** word);   // of the current device, for calls without a status word
cudaError_t launch_q8_merge(const Q8Run& r, const Q8Plan& p, int64_t pair0, int pairs, const float* part, const float* part_lse,
                            cudaStream_t st);
cudaError_t launch_attention_q8(const Q8Run& r, const Q8Plan& p, void* workspace, cudaStream_t st);

}  // namespace tq
