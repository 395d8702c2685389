// tq_draft.cu — trees of drafted tokens: ancestor masks and depths from the nodes' parents.
//
// A thread walks one node's way up to its root.  Parents come before their children, so the ancestors' numbers fall and
// the words of the mask are filled from the node's own downwards, each written once.  A walk has as many steps as the
// node is deep, each a read of shared memory: 16 trees of 26 nodes take the launch's time.
#include "tq_evict.h"

namespace tq {

constexpr int DRAFT_THREADS = 128;

__global__ void __launch_bounds__(DRAFT_THREADS) draft_tree_kernel(const int32_t* __restrict__ parents, int64_t stride, int n, int words,
                                                                   uint32_t* __restrict__ mask, int32_t* __restrict__ depth) {
    extern __shared__ int s_parent[];
    const int64_t b = blockIdx.y;
    const int first = blockIdx.x * DRAFT_THREADS, last = first + DRAFT_THREADS < n ? first + DRAFT_THREADS : n;
    for (int i = threadIdx.x; i < last; i += DRAFT_THREADS) {
        const int p = parents[b * stride + i];
        s_parent[i] = p >= 0 && p < i ? p : -1;   // anything else is a root
    }
    __syncthreads();
    const int i = first + threadIdx.x;
    if (i >= n) return;
    uint32_t* row = mask ? mask + (b * n + i) * words : nullptr;
    int at = words - 1, steps = -1;
    uint32_t bits = 0;
    for (int p = i; p >= 0; p = s_parent[p]) {
        ++steps;
        if (row) {
            for (; at > (p >> 5); --at, bits = 0) row[at] = bits;
            bits |= 1u << (p & 31);
        }
    }
    if (row)
        for (; at >= 0; --at, bits = 0) row[at] = bits;
    if (depth) depth[b * n + i] = steps;
}

cudaError_t launch_draft_tree(const int32_t* parents, int64_t parents_stride, int batch, int n, uint32_t* mask, int32_t* depth,
                              cudaStream_t st) {
    const dim3 grid((n + DRAFT_THREADS - 1) / DRAFT_THREADS, batch);
    draft_tree_kernel<<<grid, DRAFT_THREADS, n * sizeof(int), st>>>(parents, parents_stride, n, (n + 31) / 32, mask, depth);
    return cudaGetLastError();
}

}  // namespace tq
