// tq_select.cu — which cached tokens stay: of every (sequence, KV head) the last ones, the first ones, and of the others those
// with the largest sums of attention weights, ties to the lowest slot, in rising order.
//
// A weight's order is that of an unsigned 32-bit key.  The key of the last token that stays is found digit by digit
// from the top (11, 11 and 10 bits): the tokens that agree with the digits so far are counted by their next digit, and
// the digit is the one in which the wanted rank falls.  Then the tokens above it, and as many of its equals as are
// wanted, are written in the order of their slots, each at the count of those before it.
//
// A cluster of CTAs shares a (sequence, KV head): each takes a run of slots and keeps its keys in shared memory, so that
// weights are read once; counts are added up over the cluster's shared memories.  What bounds it: the weights' bytes take
// little time (16 x 8 heads of 32768 tokens: 17 MB); the rest is the chain of four passes with a barrier of the cluster after
// each.  11 bits take the sign, the exponent and two bits of the fraction, so that weights of like size, which most are,
// do not meet in one counter.
#include <cooperative_groups.h>

#include "leankv_tq.h"
#include "tq_evict.h"
#include "tq_kernels.h"

namespace cg = cooperative_groups;

namespace tq {

constexpr int SEL_THREADS = 512, SEL_WARPS = SEL_THREADS / 32, SEL_BINS = 2048;
constexpr int SEL_MOST = 8;                          // CTAs of a cluster
constexpr int SEL_KEYS = 40 * 1024;                  // keys that a CTA can keep
constexpr int SEL_GROUP = SEL_THREADS;               // slots of a CTA come in multiples of this

// larger weights have larger keys; NaN counts as -inf, -0 as 0; 0 is below all of them
__device__ __forceinline__ uint32_t weight_key(float w) {
    uint32_t u = __float_as_uint(w);
    if (u == 0x80000000u) u = 0u;
    if (w != w) u = 0xFF800000u;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct SelectShared {
    uint32_t bins[3][SEL_BINS];
    uint32_t warp_sums[SEL_WARPS];
    uint32_t over[SEL_WARPS], same[SEL_WARPS];       // of a warp's slots: above the border, at it
    uint32_t totals[2];                              // of the CTA
    uint32_t digit, left;
};

// CACHED: keys are kept in shared memory; else (more slots than a cluster holds) weights are read in every pass
template <bool CACHED>
__global__ void __launch_bounds__(SEL_THREADS) select_kernel(const SelectRun r, int per_cta) {
    extern __shared__ uint32_t s_keys[];
    __shared__ SelectShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int64_t pair = blockIdx.x / size;
    const int h = (int)(pair % r.Hkv), b = (int)(pair / r.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t cap = r.max_pages << r.page_shift;
    int64_t len64 = r.kv_len[b];
    len64 = len64 < 0 ? 0 : (len64 > cap ? cap : len64);
    if (len64 > r.max_len) {
        len64 = r.max_len;
        if (threadIdx.x == 0 && r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
    }
    const int len = (int)len64;
    int64_t keep64 = r.keep ? r.keep[b] : r.width;
    keep64 = keep64 < 0 ? 0 : (keep64 > r.width ? r.width : keep64);
    const int k = (int)(keep64 < len ? keep64 : len);
    const int recent = (int)(r.recent < k ? r.recent : k), sinks = (int)(r.sinks < k - recent ? r.sinks : k - recent);
    const int lo = sinks, hi = len - recent;           // candidates [lo, hi)
    const uint32_t want = (uint32_t)(k - recent - sinks);
    int32_t* out = r.slots + pair * r.width;
    // the fixed ones, and -1 behind the last
    for (int64_t i = (int64_t)rank * SEL_THREADS + threadIdx.x; i < r.width; i += (int64_t)size * SEL_THREADS) {
        if (i < sinks) out[i] = (int)i;
        else if (i >= k) out[i] = -1;
        else if (i >= k - recent) out[i] = hi + (int)(i - (k - recent));
    }
    if (want == 0) return;                             // for all CTAs of the cluster

    const int begin = rank * per_cta;                  // this CTA's slots, a warp's run of them
    const int per_warp = per_cta / SEL_WARPS, w0 = begin + warp * per_warp;
    const float* pool = r.weights;
    const int32_t* pages = r.pages + (int64_t)b * r.max_pages;
    const int in_page = (1 << r.page_shift) - 1;
    auto load = [&](int slot) -> uint32_t {
        const int32_t pg = pages[slot >> r.page_shift];
        if (pg < 0 || pg >= r.num_pages) {             // holds nothing: goes before all others
            if (r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
            return 0u;
        }
        return weight_key(pool[((((int64_t)pg * r.Hkv + h) << r.page_shift)) + (slot & in_page)]);
    };
    for (int i = threadIdx.x; i < 3 * SEL_BINS; i += SEL_THREADS) sh.bins[0][i] = 0;
    __syncthreads();
    uint32_t border = 0, left = want;                  // digits found so far; rank among those that agree with them
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        uint32_t* bins = sh.bins[pass];
        for (int i = lane; i < per_warp; i += 32) {
            const int slot = w0 + i;
            if (slot >= hi) break;
            uint32_t key;
            if (pass == 0 || !CACHED) {
                if (slot < lo) continue;
                key = load(slot);
                if (CACHED) s_keys[slot - begin] = key;
            } else {
                if (slot < lo) continue;
                key = s_keys[slot - begin];
            }
            if (pass == 0 || (key >> (shift + bits)) == (border >> (shift + bits))) atomicAdd(bins + ((key >> shift) & ((1u << bits) - 1)), 1u);
        }
        cluster.sync();
        // bins from the top: a thread has four of them
        const int at = SEL_BINS - 4 - 4 * threadIdx.x;
        uint4 sum = make_uint4(0, 0, 0, 0);
        for (int c = 0; c < size; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(bins, c) + at);
            sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
        }
        uint32_t before = sum.x + sum.y + sum.z + sum.w;
        const uint32_t mine = before;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        if (lane == 31) sh.warp_sums[warp] = before;
        __syncthreads();
        before -= mine;
        for (int w = 0; w < warp; ++w) before += sh.warp_sums[w];
        if (before < left && before + mine >= left) {
            uint32_t x[4] = {sum.w, sum.z, sum.y, sum.x};
            int d = 0;
            while (d < 3 && before + x[d] < left) before += x[d++];
            sh.digit = (uint32_t)(at + 3 - d);
            sh.left = left - before;
        }
        __syncthreads();
        border |= sh.digit << shift;
        left = sh.left;
    }

    // those above the border all stay, and the first `left` of those at it
    uint32_t over = 0, same = 0;
    for (int i = lane; i < per_warp; i += 32) {
        const int slot = w0 + i;
        if (slot >= hi) break;
        if (slot < lo) continue;
        const uint32_t key = CACHED ? s_keys[slot - begin] : load(slot);
        over += key > border;
        same += key == border;
    }
    over = __reduce_add_sync(0xffffffffu, over);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) {
        sh.over[warp] = over;
        sh.same[warp] = same;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        uint32_t t = 0;
        for (int w = 0; w < SEL_WARPS; ++w) t += threadIdx.x ? sh.same[w] : sh.over[w];
        sh.totals[threadIdx.x] = t;
    }
    cluster.sync();
    over = same = 0;                                   // before this warp's slots
    for (int c = 0; c < rank; ++c) {
        const uint32_t* t = cluster.map_shared_rank(sh.totals, c);
        over += t[0];
        same += t[1];
    }
    for (int w = 0; w < warp; ++w) {
        over += sh.over[w];
        same += sh.same[w];
    }
    for (int i = 0; i < per_warp && w0 + i < hi; i += 32) {
        const int slot = w0 + i + lane;
        const bool in = slot >= lo && slot < hi;
        const uint32_t key = in ? (CACHED ? s_keys[slot - begin] : load(slot)) : 0u;
        const uint32_t up = __ballot_sync(0xffffffffu, in && key > border), eq = __ballot_sync(0xffffffffu, in && key == border);
        const uint32_t below = (1u << lane) - 1;
        const uint32_t o = over + __popc(up & below), e = same + __popc(eq & below);
        const bool stays = ((up >> lane) & 1) || (((eq >> lane) & 1) && e < left);
        if (stays) out[sinks + o + (e < left ? e : left)] = slot;
        over += __popc(up);
        same += __popc(eq);
    }
    cluster.sync();                                    // no CTA ends while another one may still read its shared memory
}

cudaError_t launch_select(const SelectRun& r, cudaStream_t st) {
    const int64_t pairs = (int64_t)r.B * r.Hkv;
    // CTAs of a (sequence, KV head): as many as are resident together (three a SM by their threads and bins), none with
    // fewer than 2048 slots to look at, since each adds to the counting over the cluster
    int size = 1;
    while (size < SEL_MOST && pairs * size * 2 <= 3 * (int64_t)sm_count() && r.max_len > size * 2048) size *= 2;
    while (size < SEL_MOST && r.max_len > (int64_t)size * SEL_KEYS) size *= 2;
    const int64_t per64 = ((r.max_len + size - 1) / size + SEL_GROUP - 1) / SEL_GROUP * SEL_GROUP;
    const int per = (int)per64;
    const bool cached = per <= SEL_KEYS;
    if (pairs * size >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(pairs * size));
    cfg.blockDim = dim3(SEL_THREADS);
    cfg.dynamicSmemBytes = cached ? (size_t)per * sizeof(uint32_t) : 0;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!cached) return cudaLaunchKernelEx(&cfg, select_kernel<false>, r, per);
    const cudaError_t e = cudaFuncSetAttribute(select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_KEYS * (int)sizeof(uint32_t));
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, select_kernel<true>, r, per);
}

}  // namespace tq
