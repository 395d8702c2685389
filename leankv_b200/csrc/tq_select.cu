// tq_select.cu — which cached tokens stay: of every (sequence, KV head) the last ones, the first ones, and of the others those
// with the largest sums of attention weights, ties to the lowest slot, in rising order.
//
// A weight's order is that of an unsigned 32-bit key.  The key of the last token that stays is found digit by digit
// from the top (11, 11 and 10 bits): the tokens that agree with the digits so far are counted by their next digit, and
// the digit is the one in which the wanted rank falls.  Then the tokens above it, and as many of its equals as are
// wanted, are written in the order of their slots, each at the count of those before it.
//
// A CTA keeps the keys of up to 32768 slots, 32 a thread, so that weights are read once: in registers, but 28 words of a thread's
// (112 bytes stored, 128 loaded), which 64 registers for each of 1024 threads do not hold.  Its counters are in shared memory.
// Where sequences are longer, or there are few (sequence, KV head)s, a cluster of CTAs shares one, and counts are added up over
// their shared memories; a barrier of the cluster costs about as much as a pass over 8192 keys (128 of them of 32768 slots: 36 us
// in clusters of two, 48 and 110 us in clusters of four and eight).  What bounds it: the chain of four passes, counting by atomics
// and barriers; the weights' bytes take little time (16 x 8 heads of 32768 tokens, 17 MB: 20 us, floor 3; issue 61 %, integer pipe
// 55 %; 42 us when every pass read them again).  Weights that are all alike, whose counting meets in one word: 19 us.  One sequence
// of 1025 tokens: 6.5 us.  11 bits take the sign, the exponent and two bits of the fraction, so that weights of like size, which
// most are, do not meet in one counter.
#include <cooperative_groups.h>

#include "leankv_tq.h"
#include "tq_evict.h"
#include "tq_kernels.h"

namespace cg = cooperative_groups;

namespace tq {

constexpr int SEL_THREADS = 1024, SEL_WARPS = 32, SEL_BINS = 2048;
constexpr int SEL_MOST = 8;                          // CTAs of a cluster
constexpr int SEL_KEYS = 32;                         // keys that a thread can keep
constexpr int SEL_SHARE = 8192;                      // slots that make a CTA of a cluster worth its barriers
constexpr int SEL_BATCH = 4;                         // fours of weights of a thread that are under way together

// larger weights have larger keys; NaN counts as -inf, -0 as 0.  Below all of them are KEY_LOST (of a page outside the pool) and
// 0 (no candidate: counted with the lowest bin or not at all, and never reached from the top)
constexpr uint32_t KEY_LOST = 1;
__device__ __forceinline__ uint32_t weight_key(float w) {
    uint32_t u = __float_as_uint(w);
    if (u == 0x80000000u) u = 0u;
    if (w != w) u = 0xFF800000u;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct SelectShared {
    uint32_t bins[3 * SEL_BINS];
    uint32_t warp_sums[3][SEL_WARPS];
    uint32_t over[SEL_WARPS], same[SEL_WARPS];       // of a warp's slots: above the border, at it
    uint32_t totals[2];                              // of the CTA
    uint32_t digit[3], left[3];
};

// the sum of the values of the lanes before this one, and of all
__device__ __forceinline__ uint32_t before_lane(uint32_t x, uint32_t* all) {
    uint32_t y = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
        if ((threadIdx.x & 31) >= o) y += z;
    }
    *all = __shfl_sync(0xffffffffu, y, 31);
    return y - x;
}

// KPT: keys of a thread, a multiple of 4; 0: more slots than a cluster keeps, weights are read in every pass
template <int KPT>
__global__ void __launch_bounds__(SEL_THREADS, 1) select_kernel(const SelectRun r, int per_warp) {
    __shared__ __align__(16) SelectShared sh;
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

    // this warp's run of slots, 128 at a time, four consecutive ones (of one page) a lane
    const int64_t w64 = ((int64_t)rank * SEL_WARPS + warp) * per_warp;
    const int w0 = (int)(w64 < hi ? w64 : hi);
    const int turns = KPT ? KPT / 4 : ((hi - w0 < per_warp ? hi - w0 : per_warp) + 127) >> 7;
    const float* pool = r.weights + ((int64_t)h << r.page_shift);
    const int32_t* pages = r.pages + (int64_t)b * r.max_pages;
    const int in_page = (1 << r.page_shift) - 1;
    const int64_t page_step = (int64_t)r.Hkv << r.page_shift;
    uint32_t keys[KPT ? KPT : 1];
    // f(turn, four keys) for `n` turns of the warp from i0 on, weights as they come from memory: SEL_BATCH a lane under way together,
    // pages first
    auto read = [&](int i0, int n, auto f) {
        int32_t pg[SEL_BATCH];
        float4 w[SEL_BATCH];
#pragma unroll
        for (int u = 0; u < SEL_BATCH; ++u) {
            const int slot = w0 + 128 * (i0 + u) + 4 * lane;
            pg[u] = -2;
            if (u < n && slot + 3 >= lo && slot < hi) pg[u] = pages[slot >> r.page_shift];
        }
#pragma unroll
        for (int u = 0; u < SEL_BATCH; ++u)
            if (pg[u] >= 0 && pg[u] < r.num_pages)
                w[u] = *reinterpret_cast<const float4*>(pool + pg[u] * page_step + ((w0 + 128 * (i0 + u) + 4 * lane) & in_page));
#pragma unroll
        for (int u = 0; u < SEL_BATCH; ++u) {
            if (u >= n) continue;
            uint32_t key[4] = {0, 0, 0, 0};
            if (pg[u] >= 0 && pg[u] < r.num_pages) {
                key[0] = weight_key(w[u].x); key[1] = weight_key(w[u].y);
                key[2] = weight_key(w[u].z); key[3] = weight_key(w[u].w);
            } else if (pg[u] != -2) {
                key[0] = key[1] = key[2] = key[3] = KEY_LOST;
                if (r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
            }
            const int slot = w0 + 128 * (i0 + u) + 4 * lane;
            if (slot < lo || slot + 3 >= hi) {   // the ends of the candidates
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (slot + v < lo || slot + v >= hi) key[v] = 0;
            }
            f(i0 + u, key);
        }
    };
    auto every = [&](auto f) {
        if constexpr (KPT > 0) {
#pragma unroll
            for (int i = 0; i < KPT / 4; ++i) f(i, keys + 4 * i);
        } else {
            for (int i = 0; i < turns; i += SEL_BATCH) read(i, turns - i, f);
        }
    };
    for (int i = threadIdx.x; i < 3 * SEL_BINS; i += SEL_THREADS) sh.bins[i] = 0;
    if constexpr (KPT > 0) {
#pragma unroll
        for (int i0 = 0; i0 < KPT / 4; i0 += SEL_BATCH)
            read(i0, KPT / 4 - i0, [&](int i, const uint32_t* key) {
#pragma unroll
                for (int v = 0; v < 4; ++v) keys[4 * i + v] = key[v];
            });
    }
    __syncthreads();
    uint32_t border = 0, left = want;                  // digits found so far; rank among those that agree with them
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        uint32_t* bins = sh.bins + pass * SEL_BINS;
        every([&](int, const uint32_t* key) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (pass == 0 ? key[v] != 0 : (key[v] >> (shift + bits)) == (border >> (shift + bits)))
                    atomicAdd(bins + (pass == 0 ? key[v] >> shift : (key[v] >> shift) & ((1u << bits) - 1)), 1u);
        });
        // bins from the top: a thread has two of them
        const int at = SEL_BINS - 2 - 2 * threadIdx.x;
        uint2 sum;
        if (size > 1) {
            cluster.sync();
            sum = make_uint2(0, 0);
            for (int c = 0; c < size; ++c) {
                const uint2 x = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(bins, c) + at);
                sum.x += x.x; sum.y += x.y;
            }
        } else {
            __syncthreads();
            sum = *reinterpret_cast<const uint2*>(bins + at);
        }
        const uint32_t mine = sum.x + sum.y;
        uint32_t all, before = before_lane(mine, &all);
        if (lane == 31) sh.warp_sums[pass][warp] = all;
        __syncthreads();
        uint32_t rest;
        const uint32_t others = before_lane(sh.warp_sums[pass][lane], &rest);
        before += __shfl_sync(0xffffffffu, others, warp);
        if (before < left && before + mine >= left) {
            const bool second = before + sum.y < left;   // the upper bin does not reach
            sh.digit[pass] = (uint32_t)(at + (second ? 0 : 1));
            sh.left[pass] = left - before - (second ? sum.y : 0);
        }
        __syncthreads();
        border |= sh.digit[pass] << shift;
        left = sh.left[pass];
    }

    // those above the border all stay, and the first `left` of those at it
    uint32_t over = 0, same = 0;
    every([&](int, const uint32_t* key) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            over += key[v] > border;
            same += key[v] == border;
        }
    });
    over = __reduce_add_sync(0xffffffffu, over);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) {
        sh.over[warp] = over;
        sh.same[warp] = same;
    }
    __syncthreads();
    // before this warp's slots
    uint32_t all_over, all_same;
    const uint32_t o32 = before_lane(sh.over[lane], &all_over), s32 = before_lane(sh.same[lane], &all_same);
    over = __shfl_sync(0xffffffffu, o32, warp);
    same = __shfl_sync(0xffffffffu, s32, warp);
    if (size > 1) {
        if (threadIdx.x == 0) {
            sh.totals[0] = all_over;
            sh.totals[1] = all_same;
        }
        cluster.sync();
        for (int c = 0; c < rank; ++c) {
            const uint32_t* t = cluster.map_shared_rank(sh.totals, c);
            over += t[0];
            same += t[1];
        }
    }
    int32_t* at = out + sinks;
    every([&](int i, const uint32_t* key) {
        // tokens above the border and at it, in the lanes before and in this one (16 bits each: at most 128)
        uint32_t mine = 0;
#pragma unroll
        for (int v = 0; v < 4; ++v) mine += (key[v] > border ? 1u : 0u) + (key[v] == border ? 0x10000u : 0u);
        uint32_t all, o = before_lane(mine, &all), e = same + (o >> 16);
        o = over + (o & 0xFFFFu);
        const int slot = w0 + 128 * i + 4 * lane;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const bool up = key[v] > border, eq = key[v] == border;
            if (up || (eq && e < left)) at[o + (e < left ? e : left)] = slot + v;
            o += up;
            e += eq;
        }
        over += all & 0xFFFFu;
        same += all >> 16;
    });
    if (size > 1) cluster.sync();                      // no CTA ends while another one may still read its shared memory
}

template <int KPT> static cudaError_t launch_select_k(const SelectRun& r, int size, int per_warp, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((int64_t)r.B * r.Hkv * size));
    cfg.blockDim = dim3(SEL_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, select_kernel<KPT>, r, per_warp);
}

cudaError_t launch_select(const SelectRun& r, cudaStream_t st) {
    const int64_t pairs = (int64_t)r.B * r.Hkv;
    // CTAs of a (sequence, KV head): one, but where SMs would be idle as many as look at SEL_SHARE slots each, and as many as it
    // takes to keep the keys
    int size = 1;
    while (size < SEL_MOST && pairs * size * 2 <= sm_count() && r.max_len > (int64_t)size * SEL_SHARE) size *= 2;
    while (size < SEL_MOST && r.max_len > (int64_t)size * SEL_THREADS * SEL_KEYS) size *= 2;
    if (pairs * size >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    const int64_t per = (r.max_len + size - 1) / size;       // slots of a CTA
    if (per <= 4 * SEL_THREADS) return launch_select_k<4>(r, size, 4 * 32, st);
    if (per <= 8 * SEL_THREADS) return launch_select_k<8>(r, size, 8 * 32, st);
    if (per <= SEL_KEYS * SEL_THREADS) return launch_select_k<SEL_KEYS>(r, size, SEL_KEYS * 32, st);
    return launch_select_k<0>(r, size, (int)((per + 4 * SEL_THREADS - 1) / (4 * SEL_THREADS) * 128), st);
}

}  // namespace tq
