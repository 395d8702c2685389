// tq_evict.h — internal interface of drafted trees, sums of attention weights, selection and moving of cached tokens.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "tq_attn_q8.h"

namespace tq {

// masks [batch][n][words] and depths [batch][n] (either may be null) of trees given by parents [batch][n]
cudaError_t launch_draft_tree(const int32_t* parents, int64_t parents_stride, int batch, int n, uint32_t* mask, int32_t* depth,
                              cudaStream_t st);

// Sums of attention weights: the queries, keys and pages are the Q8Run's (k: blocks of k_type).
struct WeightsRun {
    Q8Run q;
    int k_type = 8;
    const float* lse = nullptr;       // [B][Hq][n]
    int64_t window = 0;               // rows of each sequence that count, its last ones
    float decay = 1.0f;
    const int32_t* fresh = nullptr;   // slots from here on begin anew (null: none)
    float* weights = nullptr;         // [num_pages][Hkv][page]
};
struct WeightsPlan {
    int rows = 8, chunks = 1;         // query rows of a KV head at a time, and how often
    int splits = 1;                   // CTAs that share a (sequence, KV head)
    bool tensor = false;              // many rows, on tcgen05:
    int tiles = 0;                    // row tiles of a (sequence, KV head) in the work memory
    int pairs_pass = 0;               // (sequence, KV head) pairs that run at a time
    size_t bytes = 0;                 // work memory
};
// n: query tokens that count
WeightsPlan weights_plan(int B, int Hkv, int grp, int D, int64_t n, int64_t max_len, bool q8);
cudaError_t launch_weights(const WeightsRun& r, const WeightsPlan& p, void* workspace, cudaStream_t st);
void weights_rows_plan(int64_t pairs, int D, int64_t rows, int64_t len, WeightsPlan* p);
cudaError_t launch_weights_rows(const WeightsRun& r, const WeightsPlan& p, void* workspace, cudaStream_t st);

struct SelectRun {
    int B = 0, Hkv = 0;
    const float* weights = nullptr;   // [num_pages][Hkv][page]
    const int32_t* pages = nullptr;
    int64_t max_pages = 0, num_pages = 0;
    int page_shift = 4;
    const int32_t* kv_len = nullptr;
    const int32_t* keep = nullptr;    // null: width
    int64_t width = 0, sinks = 0, recent = 0;
    int max_len = 0;
    int32_t* slots = nullptr;         // [B][Hkv][width]
    int32_t* status = nullptr;
};
cudaError_t launch_select(const SelectRun& r, cudaStream_t st);

struct MoveSide {
    uint8_t* pool = nullptr;
    float* scale = nullptr;           // 8-bit pages
    int type = 8;
};
struct MoveRun {
    int B = 0, Hkv = 0, D = 0;
    int64_t n = 0;                    // rows of a (sequence, KV head)
    const int32_t* src = nullptr;     // [B][src_heads][n]
    int src_heads = 1;
    const int32_t* first = nullptr;   // null: 0
    const int32_t* count = nullptr;   // null: n
    MoveSide k, v;
    float* weights = nullptr;         // [num_pages][Hkv][page], or null
    const int32_t* from = nullptr;    // page tables
    const int32_t* to = nullptr;
    int64_t max_from = 0, max_to = 0, num_pages = 0;
    int page_shift = 4;
    bool in_place = true;
    int32_t* overflow = nullptr;
    int32_t* status = nullptr;
    uint32_t* flags = nullptr;        // a ticket, then one word per chunk (zeroed by the launch); null: one chunk each
};
int64_t move_chunks(int64_t n, bool with_first);
cudaError_t launch_move(const MoveRun& r, cudaStream_t st);

}  // namespace tq
