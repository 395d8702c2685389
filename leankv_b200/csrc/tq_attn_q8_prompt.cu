// tq_attn_q8_prompt.cu — attention over 8-bit pages for prompts and long drafts, on tcgen05.
//
// The mathematics is tq_attn_q8.cu's.  With many query rows per KV head the two products and the exponentials bound
// it, not the cache: an 8192-token causal prompt of 32 heads of 128 (550 Gflop with the masked half left out) takes
// 563 to 597 us, 920 to 977 Tflop/s; the products alone would take 337 us at the measured bf16 rate, the
// exponentials (16 a cycle and SM) about as long, and a row's softmax waits for its scores and its values for its
// weights.  ncu on that case: tensor pipe 44 %, special function unit 45 %, issue 46 %.  Two ways of getting f16 tiles
// from codes, chosen by rows (q8_plan in tq_attn_q8.cu has both sides' times):
//
// tiles (DIRECT = false), many rows: expand_q8_kernel turns the codes that the rows will see into f16 tiles, once,
// in work memory: a tile is the image of its shared-memory buffer, so that the second kernel fetches it with one bulk
// copy.  (Converted by warps of the second kernel, every tile would be converted for each of a prompt's row tiles:
// 28 % of its instructions, 677 instead of 606 us for the 8192-token prompt when that was changed.)  It also gathers
// what a block's scales contribute to the scores.
//
// DIRECT, up to a few row tiles: seven warps of the attention kernel convert the codes on their way into shared
// memory (convert_tiles), with no work memory and no first pass over the cache.
//
// attn_q8_prompt_kernel: a CTA takes QT tiles of 128 query rows (tokens x heads of one group) of one (sequence, KV
// head), or one split of their tokens.  Warps:
//   8 QT softmax warps   two threads per row, half of a tile's columns each: scores from TMEM, weights back to
//                        TMEM, the output's rescaling
//   1 issuing warp       one elected lane issues all tcgen05.mma
//   1 loading warp       one lane issues the bulk copies of K and V tiles; DIRECT: 7 converting warps in its place
// Per tile of KT tokens: S = Q K^T (both from shared memory, f16, fp32 sums in TMEM), weights P in f16 written over
// S, O += P V (P from TMEM, V from shared memory).  D = 128 from tiles, where there are enough rows: two row tiles
// take turns, so that one's softmax runs while the other's products do; TMEM holds S and O of both (512 columns).
// Otherwise one row tile has two buffers for S: D = 256, whose O alone takes 256 columns and Q 64 KB, takes 64
// tokens at a time.
//
// Roundings: a row of q' is scaled by its largest element and rounded to f16, for outputs of more than bf16's 8
// bits (LO) to the sum of two f16 terms; the second one is read from TMEM.  With one term the float16 answer of 700
// rows was off by 4.3e-4 of its norm, with two by 2.8e-4 (2.1e-4 is float16's own rounding); the time rises by the
// products, 118 -> 136 us for pieces of prompts of heads of 256, 597 -> 753 us for the 8192-token prompt.  In
// bfloat16, off by 1.7e-3 either way, the second term is left out.  Weights are f16, off by up to 2^-11 of each,
// which averages out over the tokens.
//
// Tiles are runs of 64 elements: [row][128 bytes], 16-byte chunk c of row x at c ^ (x & 7) (the 128-byte
// swizzle of the matrix descriptors).  K is read with its elements contiguous, V as the transposed operand from
// the same layout.  Codes are exact in f16; scales never touch the tiles: they enter with the scores.
//
// Every wait gives up after about a second (status TQ_ERROR_TIMEOUT) instead of hanging; copies and products that were
// issued before are waited for (tq_wait.h).
#include "leankv_tq.h"
#include "tq_attn_q8.cuh"
#include "tq_kernels.h"
#include "tq_tc.cuh"

#include <type_traits>

namespace tq {

// DIRECT: codes are converted by warps of the kernel itself
// QTILES: row tiles of a CTA; two only with D = 128 from tiles
template <int D, bool DIRECT, int QTILES> struct PromptCfg {
    static constexpr int QT = QTILES, KT = D == 128 ? 128 : 64, ROWS = 128 * QT;
    static constexpr int LO_COL = D == 128 ? 384 : 128;
    static constexpr int SEGS = D / 64;                    // 64-element runs of a row
    static constexpr int Q_TILE = 128 * D * 2, KV_TILE = KT * D * 2, SEG = KT * 128;
    static constexpr int SBUF = 2;                         // S buffers: one per row tile, or two of one
    static constexpr int TPR = 2;                          // softmax threads per row
    static constexpr int SOFT_WARPS = 4 * TPR * QT, ISSUE = SOFT_WARPS, LOAD = SOFT_WARPS + 1;
    static constexpr int CONV_WARPS = 7, WARPS = LOAD + (DIRECT ? CONV_WARPS : 1);
    static constexpr int COLS = KT / TPR;                  // columns of a softmax thread
    static constexpr int BPT = KT / 16;                    // scale blocks of a tile
    static constexpr int TILES = QT * Q_TILE + 4 * KV_TILE;   // Q, two K and two V buffers
    static constexpr int SMEM = TILES + 1024;              // the tiles start on 1024 bytes
};

// a block's factors from its scales (blk -1: not there)
__device__ __forceinline__ float4 block_factors(int blk, float ks, float vs) {
    if (blk < 0) return make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
    const float vse = vs > 0.0f ? vs : Q8_ZERO_SCALE;
    return make_float4(ks, lg2(vse), __frcp_rn(vse), 0.0f);
}

// ── codes to tiles ─────────────────────────────────────────────────────────
// Work memory of the pairs (sequence, KV head) of one pass: K and V tiles [pair][tile][2][KV_TILE bytes], then the
// blocks' factors [pair][tile][BPT] as float4 (K scale, log2 and reciprocal of the V scale): a score enters the
// softmax as s * factor.x + factor.y, its weight counts factor.z.  Blocks that are not there (behind the last
// token, pages outside the pool) get a log2 of -inf: their weights are 0.
template <int D>
__global__ void __launch_bounds__(256) expand_q8_kernel(const Q8Run r, int64_t pair0, int tiles_max, uint8_t* __restrict__ tiles,
                                                        float4* __restrict__ factors) {
    using C = PromptCfg<D, false, 1>;   // the same with two row tiles
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tile = blockIdx.x % tiles_max;
    const int64_t slot = blockIdx.x / tiles_max, pair = pair0 + slot;
    const int h = (int)(pair % r.Hkv), b = (int)(pair / r.Hkv);
    const SeqLens sl = seq_lens(r, b);
    if (tile * C::KT >= sl.len || sl.q_len == 0) return;   // tile < tiles_max by the grid
    uint8_t* image = tiles + (slot * tiles_max + tile) * (2 * C::KV_TILE);
    // a warp takes 8 rows x 64 elements (four lanes a row, 16 codes a lane) at a time
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane >> 2, c4 = lane & 3;
#pragma unroll
    for (int i = 0; i < C::KT / 8 * C::SEGS / 8; ++i) {
        const int u = warp + 8 * i, seg = u % C::SEGS, row = u / C::SEGS * 8 + sub;
        const int tok = tile * C::KT + row;
        const int blk = (tok & ~15) < sl.len ? block_at(r, b, h, tok >> 4) : -1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (blk >= 0)
                w = __ldg(reinterpret_cast<const uint4*>((x ? r.v : r.k) + ((int64_t)blk * 16 + (tok & 15)) * D + seg * 64 + 16 * c4));
            uint32_t o[8];
            codes_to_f16(w, o);
            uint8_t* to = image + x * C::KV_TILE + seg * C::SEG + row * 128;
            *reinterpret_cast<uint4*>(to + (((2 * c4) ^ sub) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(to + (((2 * c4 + 1) ^ sub) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
    if (threadIdx.x < C::BPT) {
        const int block = tile * C::BPT + threadIdx.x;
        int blk = -1;
        if (block * 16 < sl.len) {
            blk = block_at(r, b, h, block);
            if (blk < 0 && r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
        }
        const float4 f = block_factors(blk, blk < 0 ? 0.0f : r.ks[blk], blk < 0 ? 0.0f : r.vs[blk]);
        factors[(slot * tiles_max + tile) * C::BPT + threadIdx.x] = f;
    }
}

// ── conversion by warps of the attention kernel (DIRECT) ────────────────────
// A tile of K or V is 16 units of a 16-token block and 64 elements (1 KB of codes, two 16-byte loads and four
// stores a lane); warp cw takes units cw, cw + 7, cw + 14.  K and V of a tile follow one another; codes are loaded
// one tensor ahead, pages two tiles ahead.  Warp 0 also provides the blocks' factors.
template <int D>
__device__ __forceinline__ void convert_tiles(const Q8Run& r, int b, int h, int t_begin, int tiles_n, int kv_end, int cw,
                                              uint32_t k_at, uint32_t v_at, uint32_t k_full, uint32_t k_empty,
                                              uint32_t v_full, uint32_t v_empty, float4 (*s_fac)[PromptCfg<D, true, 1>::BPT],
                                              uint32_t f_full, volatile int* failed) {
    using C = PromptCfg<D, true, 1>;
    constexpr int NU = 3;
    const int lane = threadIdx.x & 31, sub = lane >> 2, c4 = lane & 3, per_page = r.page_shift - 4;
    const int32_t* pages = r.pages + (int64_t)b * r.max_pages;
    // lanes 0 .. 2: the page of unit cw + 7 lane; lanes 8 .. : that of block lane - 8 (for the factors)
    int page = -1;
    auto lane_block = [&](int t) { return (t_begin + t) * C::BPT + (lane < 8 ? (cw + 7 * lane) / C::SEGS : lane - 8); };
    auto load_page = [&](int t) {
        const int block = lane_block(t);
        page = -2;   // none
        if ((lane < 8 ? cw + 7 * lane < 16 : cw == 0 && lane - 8 < C::BPT) && t < tiles_n && block * 16 < kv_end)
            page = pages[block >> per_page];
    };
    int at[NU], fac_blk = -1;      // blocks of the units (-1: no tokens there) and of the lane's factors
    float fac_ks = 0.0f, fac_vs = 0.0f;
    auto locate = [&](int t) {
        const int block = lane_block(t);
        int blk = -1;
        if (page >= 0 && page < r.num_pages) blk = ((page * r.Hkv + h) << per_page) + (block & ((1 << per_page) - 1));
        else if (page != -2 && r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
#pragma unroll
        for (int i = 0; i < NU; ++i) at[i] = __shfl_sync(0xffffffffu, blk, i);
        if (cw == 0 && lane >= 8) {
            fac_blk = blk;
            if (blk >= 0) {
                fac_ks = r.ks[blk];
                fac_vs = r.vs[blk];
            }
        }
    };
    auto load = [&](const int8_t* __restrict__ pool, uint4 (&w)[NU][2]) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
            if (at[i] >= 0) {
                const int8_t* p = pool + (int64_t)at[i] * (16 * D) + ((cw + 7 * i) % C::SEGS) * 64 + sub * D + 16 * c4;
                w[i][0] = ldg_now(p);
                w[i][1] = ldg_now(p + 8 * D);
            }
        }
    };
    auto store = [&](uint32_t tile, const uint4 (&w)[NU][2]) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = cw + 7 * i;
            if (u >= 16) break;
            const uint32_t to = tile + (u % C::SEGS) * C::SEG + (u / C::SEGS) * 2048 + sub * 128;
#pragma unroll
            for (int x = 0; x < 2; ++x) {   // rows sub and sub + 8 of the block
                uint32_t o[8];
                codes_to_f16(w[i][x], o);
                sts128(to + x * 1024 + (((2 * c4) ^ sub) << 4), o[0], o[1], o[2], o[3]);
                sts128(to + x * 1024 + (((2 * c4 + 1) ^ sub) << 4), o[4], o[5], o[6], o[7]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    };
    uint4 kw[NU][2], vw[NU][2];
    load_page(0);
    locate(0);
    load_page(1);
    load(r.k, kw);
    for (int t = 0; t < tiles_n; ++t) {
        const int buf = t & 1, par = ((t >> 1) & 1) ^ 1;   // the first pass over the two buffers does not wait
        load(r.v, vw);
        if (t >= 2 && !__all_sync(0xffffffffu, mbar_wait(k_empty + 8 * buf, par, failed))) break;
        if (cw == 0) {
            // ring of four: a K buffer is free again when the softmax is three tiles back
            if (lane >= 8 && lane < 8 + C::BPT) s_fac[t & 3][lane - 8] = block_factors(fac_blk, fac_ks, fac_vs);
            __syncwarp();
            if (lane == 0) mbar_arrive(f_full + 8 * (t & 3));
        }
        store(k_at + buf * C::KV_TILE, kw);
        if (lane == 0) mbar_arrive(k_full + 8 * buf);
        if (t + 1 < tiles_n) {
            locate(t + 1);
            load_page(t + 2);
            load(r.k, kw);
        }
        if (t >= 2 && !__all_sync(0xffffffffu, mbar_wait(v_empty + 8 * buf, par, failed))) break;
        store(v_at + buf * C::KV_TILE, vw);
        if (lane == 0) mbar_arrive(v_full + 8 * buf);
    }
}

// LO: q' as the sum of two f16 terms, the second one in TMEM (D / 2 columns, for which two row tiles leave no room)
// TREE: rows see what their nodes' masks say
template <int D, bool DIRECT, int QTILES, bool LO, bool TREE>
__global__ void __launch_bounds__(PromptCfg<D, DIRECT, QTILES>::WARPS * 32, 1)
attn_q8_prompt_kernel(const Q8Run r, int64_t pair0, int pairs, int tiles_max, const uint8_t* __restrict__ kv_tiles,
                      const float4* __restrict__ factors, int row_tiles, int splits, float* __restrict__ part,
                      float* __restrict__ part_lse) {
    using C = PromptCfg<D, DIRECT, QTILES>;
    constexpr int QT = C::QT, KT = C::KT, TPR = C::TPR, ROWS = C::ROWS, LPR = D / 16, THREADS = C::WARPS * 32;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[20];
    __shared__ float s_f[ROWS], s_lse[ROWS], s_top[TPR == 2 ? 2 : 1][TPR == 2 ? ROWS : 1], s_sum[TPR == 2 ? 2 : 1][TPR == 2 ? ROWS : 1];
    __shared__ __align__(16) float4 s_fac[4][C::BPT];   // blocks' factors of four tiles
    __shared__ int s_lim[ROWS];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t tile0 = smem_u32(tiles);
    const uint32_t q_at = tile0, k_at = tile0 + QT * C::Q_TILE, v_at = k_at + 2 * C::KV_TILE;
    const uint32_t bar0 = smem_u32(bars);
    const uint32_t k_full = bar0, k_empty = bar0 + 16, v_full = bar0 + 32, v_empty = bar0 + 48;   // two each
    const uint32_t s_full = bar0 + 64, p_full = bar0 + 80, o_done = bar0 + 96, done = bar0 + 104;
    const uint32_t f_full = bar0 + 112, turn = bar0 + 144;   // four, two

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // units with the most tokens first: the last row tiles of a causal prompt see the longest prefix
    const int split = blockIdx.x % splits;
    const int64_t u = blockIdx.x / splits;
    const int rt = row_tiles - 1 - (int)(u / pairs), slot = (int)(u % pairs);
    const int64_t pair = pair0 + slot;
    const int h = (int)(pair % r.Hkv), b = (int)(pair / r.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const SeqLens sl = seq_lens(r, b);
    const int total_rows = (int)r.n * r.grp, row0 = rt * ROWS;
    int last_i = (row0 + ROWS - 1) / r.grp;
    if (last_i >= sl.q_len) last_i = sl.q_len - 1;
    const int first_i = row0 / r.grp;
    int kv_end = last_i < first_i ? 0 : TREE ? sl.len : last_seen(r, sl, last_i) + 1;
    if (!DIRECT && kv_end > r.max_len) {   // longer than the caller's bound: the work memory has no tiles for it
        kv_end = r.max_len;
        if (threadIdx.x == 0 && r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
    }
    const int all_tiles = (kv_end + KT - 1) / KT, per = (all_tiles + splits - 1) / splits;
    const int t_begin = split * per < all_tiles ? split * per : all_tiles;
    const int tiles_n = all_tiles - t_begin < per ? all_tiles - t_begin : per;
    const int64_t unit = (int64_t)slot * row_tiles + rt;   // its partial rows in the work memory of this pass
    if (tiles_n <= 0 && splits > 1) {
        asm volatile("griddepcontrol.wait;" ::: "memory");   // this grid does not end before the tiles' kernel
        for (int i = threadIdx.x; i < ROWS; i += THREADS) part_lse[(unit * splits + split) * ROWS + i] = -INFINITY;
        return;
    }

    if (threadIdx.x == 0) {
        s_failed = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, DIRECT ? C::CONV_WARPS : 1);   // converting warps; or the loading lane (and bytes)
            mbar_init(v_full + 8 * i, DIRECT ? C::CONV_WARPS : 1);
            mbar_init(k_empty + 8 * i, 1);    // commits of the issuing thread
            mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4 * TPR);   // the warps of a row tile
            mbar_init(turn + 8 * i, 4 * TPR);     // the other tile's warps
        }
        for (int i = 0; i < 4; ++i) mbar_init(f_full + 8 * i, 1);
        mbar_init(o_done, 1);
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C::ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }

    // ── q': Hadamard, row maximum, f16, swizzled tiles ──
    for (int base = warp * (32 / LPR); base < ROWS; base += C::WARPS * (32 / LPR)) {
        const int row = base + lane / LPR, e0 = (lane % LPR) * 16, gr = row0 + row, i = gr / r.grp;
        const bool live = gr < total_rows && i < sl.q_len;
        float v[16];
        if (live) {
            load_row16(r.q_dtype, r.q, b * r.qs[0] + (h * r.grp + gr % r.grp) * r.qs[1] + (int64_t)i * r.qs[2] + e0, v);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.0f;
        }
        if (r.rotate_q) fwht16<D>(v, r.norm);
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
        for (int o = 1; o < LPR; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float inv = top >= 0x1p-100f ? __fdiv_rn(1.0f, top) : 0.0f;
        if (r.sm_scale < 0.0f) inv = -inv;   // the row's factor is not negative
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] *= inv;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = pack_h2(v[2 * j], v[2 * j + 1]);
        const int qt = row >> 7, rr = row & 127, c = (e0 & 63) >> 3;
        uint8_t* at = tiles + qt * C::Q_TILE + (e0 >> 6) * (128 * 128) + rr * 128;
        *reinterpret_cast<uint4*>(at + ((c ^ (rr & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(at + (((c + 1) ^ (rr & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
        if constexpr (LO) {   // what the rounding left goes to TMEM by way of the K and V buffers
            static_assert(QT * C::Q_TILE <= 4 * C::KV_TILE, "the second terms' way into TMEM");
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                w[j] = pack_h2(v[2 * j] - hi.x, v[2 * j + 1] - hi.y);
            }
            at += QT * C::Q_TILE;
            *reinterpret_cast<uint4*>(at + ((c ^ (rr & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(at + (((c + 1) ^ (rr & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        if (lane % LPR == 0) {
            s_f[row] = top * fabsf(r.sm_scale) * LOG2E;
            if constexpr (TREE) s_lim[row] = live ? last_before(sl, i) : -2;
            else s_lim[row] = live ? last_seen(r, sl, i) : -1;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the tiles are there
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    const uint32_t o_col = 256;   // S buffers at columns 0 and KT, O from 256 on
    if constexpr (LO) {
        if (warp < C::SOFT_WARPS) {   // a thread takes half a row, a run of 64 elements at a time
            static_assert(QT == 1, "one row tile's second term has room");
            const int half = (warp >> 2) & 1, rr = (warp & 3) * 32 + lane;
            const uint8_t* from = tiles + C::Q_TILE + rr * 128;
            const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + C::LO_COL;
#pragma unroll
            for (int seg = half * (C::SEGS / 2); seg < (half + 1) * (C::SEGS / 2); ++seg) {
                uint32_t x[32];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint4 y = *reinterpret_cast<const uint4*>(from + seg * (128 * 128) + ((c ^ (rr & 7)) << 4));
                    x[4 * c] = y.x; x[4 * c + 1] = y.y; x[4 * c + 2] = y.z; x[4 * c + 3] = y.w;
                }
                tc_st32(to + 32 * seg, x);
            }
            tc_wait_st();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // copies into these buffers come after
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    }

    if (warp < C::SOFT_WARPS) {
        // ── softmax: thread = half a row ──
        const int qt = warp / (4 * TPR), half = TPR == 2 ? (warp >> 2) & 1 : 0, row = qt * 128 + (warp & 3) * 32 + lane;
        const int pair_bar = 1 + qt * 4 + (warp & 3);   // barrier of the two warps of the same rows
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_at = lanes + o_col + qt * 128 + half * (D / TPR);
        const float f = s_f[row];
        const int lim = s_lim[row];
        constexpr float TINY = 1e-38f;   // least factor of a sum: -inf stays -inf where f or ks is zero
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        const bool idle = __all_sync(0xffffffffu, lim < (TREE ? -1 : 0));
        const uint32_t* mask = nullptr;   // TREE: the row's nodes
        int nodes = 0;
        if constexpr (TREE) {
            if (lim > -2) {
                mask = node_mask(r, b, (row0 + row) / r.grp);
                nodes = sl.q_len;
            }
        }
        constexpr int BPH = C::BPT / TPR, CH = C::COLS / 32;
        for (int t = 0; t < tiles_n; ++t) {
            const int sb = QT == 2 ? qt : (t & 1);
            const uint32_t s_at = lanes + sb * KT + half * C::COLS, p_at = lanes + sb * KT + half * (C::COLS / 2);
            const float4* fac = s_fac[t & 3] + half * BPH;   // factors of this thread's blocks
            const int tok0 = (t_begin + t) * KT + half * C::COLS;
            const bool edge = __any_sync(0xffffffffu, tok0 + C::COLS - 1 > lim);
            const uint32_t par = QT == 2 ? (t & 1) : ((t >> 1) & 1);
            ok = ok && __all_sync(0xffffffffu, mbar_wait(f_full + 8 * (t & 3), (t >> 2) & 1, &s_failed));
            ok = ok && __all_sync(0xffffffffu, mbar_wait(s_full + 8 * sb, par, &s_failed));
            tc_fence_after();
            if (idle) {   // no row of the warp sees anything: whatever the products make of them is not read
                if constexpr (QT == 2) {   // the turns are kept all the same: a tile that runs ahead would use up two of them
                    if (qt == 1 || t > 0)
                        ok = ok && __all_sync(0xffffffffu, mbar_wait(turn + 8 * qt, qt == 1 ? t & 1 : (t - 1) & 1, &s_failed));
                    if (ok && lane == 0) mbar_arrive(turn + 8 * (qt ^ 1));
                }
                if (!ok) break;
                if (lane == 0) mbar_arrive(p_full + 8 * sb);
                continue;
            }

            // the row's scores, in registers
            uint32_t raw[CH][32];
#pragma unroll
            for (int c = 0; c < CH; ++c) tc_ld32(s_at + 32 * c, raw[c]);
            tc_wait_ld(raw[0]);
#pragma unroll
            for (int c = 1; c < CH; ++c) tc_loaded(raw[c]);
            if (edge) {
                // few tiles: kept a branch (if-converted, these selects would cost every tile 2 instructions a score)
                asm volatile("" ::: "memory");
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int bl = 0; bl < 2; ++bl) {
                        const int first = tok0 + 32 * c + 16 * bl, left = lim - first;   // last column seen
                        if constexpr (TREE) {
                            const uint32_t seen = mask16(mask, r.tree_words, first - (sl.len - sl.q_len), nodes);
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (j > left && !((seen >> j) & 1)) raw[c][16 * bl + j] = 0xff800000u;   // -inf
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (j > left) raw[c][16 * bl + j] = 0xff800000u;   // -inf
                        }
                    }
            }
            // the largest exponent, from each scale block's largest sum (f and ks are not negative)
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < BPH; ++c) {
                const uint32_t* x = raw[c >> 1] + 16 * (c & 1);
                float y = max3(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
#pragma unroll
                for (int j = 3; j < 15; j += 2) y = max3(y, __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
                y = fmaxf(y, __uint_as_float(x[15]));
                const float2 fl = *reinterpret_cast<const float2*>(fac + c);
                top = fmaxf(top, fmaf(y, fmaxf(f * fl.x, TINY), fl.y));
            }
            if constexpr (TPR == 2) {
                // The row's other half has its own maximum (never NaN: that says that a wait ran out there, and
                // both halves leave here).  Past the barrier the other half has read its scores, too.
                s_top[half][row] = ok ? top : NAN;
                tc_fence_before();
                asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
                tc_fence_after();
                const float other = s_top[half ^ 1][row];
                ok = !__any_sync(0xffffffffu, !ok || other != other);
                top = fmaxf(top, other);
            }
            if (!ok) break;
            const bool move = top > m + Q8_SLACK;
            if (__any_sync(0xffffffffu, move)) {
                const float now = move ? top : m;
                const float w = move ? ex2(m - now) : 1.0f;
                m = now;
                l *= w;
                if (t > 0) {
                    // the products up to the last tile's are done: with two row tiles this tile's scores were
                    // issued after them, else their own commit says so
                    if (QT == 1) {
                        ok = __all_sync(0xffffffffu, mbar_wait(o_done, (t - 1) & 1, &s_failed));   // false: out by next tile
                        tc_fence_after();
                    }
#pragma unroll 1
                    for (int c = 0; c < D / TPR / 16; ++c) {   // this thread's columns of O
                        uint32_t x[16];
                        tc_ld16(o_at + 16 * c, x);
                        tc_wait_ld(x);
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * w);
                        tc_st16(o_at + 16 * c, x);
                    }
                }
            }
            // Weights 2^(s + log2 vs - m + SHIFT) in f16 over the scores, 32 of them in 16 columns.  The two row tiles
            // make theirs in turn: the special function unit, which bounds them, then works for one while the other
            // one's products run (left to themselves, both tiles fall into step and wait for each unit together).
            if constexpr (QT == 2) {
                if (qt == 1 || t > 0)
                    ok = __all_sync(0xffffffffu, mbar_wait(turn + 8 * qt, qt == 1 ? t & 1 : (t - 1) & 1, &s_failed));   // false: out by next tile
            }
            const float ref = m == -INFINITY ? 0.0f : Q8_SHIFT - m;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                uint32_t p[16];
                float e[32];
#pragma unroll
                for (int bl = 0; bl < 2; ++bl) {
                    const float4 fl = fac[2 * c + bl];
                    const float a = fmaxf(f * fl.x, TINY), y = fl.y + ref;
#pragma unroll
                    for (int j = 16 * bl; j < 16 * bl + 16; j += 2) {
                        const float2 x = __ffma2_rn(make_float2(__uint_as_float(raw[c][j]), __uint_as_float(raw[c][j + 1])),
                                                    make_float2(a, a), make_float2(y, y));
                        e[j] = x.x;
                        e[j + 1] = x.y;
                    }
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) e[j] = ex2(e[j]);
#pragma unroll
                for (int bl = 0; bl < 2; ++bl) {
                    float2 s0 = make_float2(0.0f, 0.0f), s1 = s0;
#pragma unroll
                    for (int j = 16 * bl; j < 16 * bl + 16; j += 4) {
                        s0 = __fadd2_rn(s0, make_float2(e[j], e[j + 1]));
                        s1 = __fadd2_rn(s1, make_float2(e[j + 2], e[j + 3]));
                    }
                    l = fmaf((s0.x + s0.y) + (s1.x + s1.y), fac[2 * c + bl].z, l);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) p[j] = pack_h2(e[2 * j], e[2 * j + 1]);
                tc_st16(p_at + 16 * c, p);
            }
            if constexpr (QT == 2) {
                __syncwarp();
                if (lane == 0) mbar_arrive(turn + 8 * (qt ^ 1));
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * sb);
        }
        if constexpr (TPR == 2) {
            s_sum[half][row] = l;
            asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
            l = s_sum[0][row] + s_sum[1][row];
        }
        if (half == 0) {
            s_lse[row] = l > 0.0f ? (m - Q8_SHIFT + lg2(l)) * LN2 : -INFINITY;
            s_f[row] = l > 0.0f ? __fdiv_rn(1.0f, l) : 0.0f;
        }
    } else if (warp == C::ISSUE) {
        // ── issue ──
        if (tiles_n > 0) {
            constexpr uint32_t id_s = mma_idesc(KT, 0), id_o = mma_idesc(D, 1);
            const uint32_t one = tc_elect();
            // descriptors count in 16 bytes; no tile crosses the address field's end
            const uint64_t q_desc = tile_desc(q_at, 16), k_desc = tile_desc(k_at, 16), v_desc = tile_desc(v_at, C::SEG);
            bool ok = true;
            auto scores = [&](int qt, int t) {
                const uint64_t q = q_desc + qt * (C::Q_TILE >> 4), k = k_desc + (t & 1) * (C::KV_TILE >> 4);
                const uint32_t d = tmem + (QT == 2 ? qt : (t & 1)) * KT;
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    tc_mma_ss(one, d, q + ((j >> 2) * (128 * 128 >> 4) + (j & 3) * 2), k + ((j >> 2) * (C::SEG >> 4) + (j & 3) * 2), id_s, j > 0);
                if constexpr (LO) {
#pragma unroll
                    for (int j = 0; j < D / 16; ++j)
                        tc_mma_ts(one, d, tmem + C::LO_COL + 8 * j, k + ((j >> 2) * (C::SEG >> 4) + (j & 3) * 2), id_s, 1);
                }
                tc_commit(one, s_full + 8 * (QT == 2 ? qt : (t & 1)));
            };
            auto values = [&](int qt, int t) {
                const uint32_t p = tmem + (QT == 2 ? qt : (t & 1)) * KT;
                const uint64_t v = v_desc + (t & 1) * (C::KV_TILE >> 4);
#pragma unroll
                for (int j = 0; j < KT / 16; ++j)
                    tc_mma_ts(one, tmem + o_col + qt * 128, p + 8 * j, v + j * 128, id_o, t > 0 || j > 0);
            };
            auto full = [&](uint32_t bar, int t) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait(bar + 8 * (t & 1), (t >> 1) & 1, &s_failed));
                tc_fence_after();
                return ok;
            };
            if constexpr (QT == 2) {
                if (full(k_full, 0)) {
                    scores(0, 0);
                    scores(1, 0);
                    tc_commit(one, k_empty);
                }
                for (int t = 0; ok && t < tiles_n; ++t) {
                    if (!full(v_full, t)) break;
                    for (int qt = 0; qt < 2; ++qt) {
                        ok = ok && __all_sync(0xffffffffu, mbar_wait(p_full + 8 * qt, t & 1, &s_failed));
                        if (!ok) break;
                        tc_fence_after();
                        values(qt, t);
                        if (qt == 1) tc_commit(one, v_empty + 8 * (t & 1));
                        if (t + 1 < tiles_n) {
                            if (qt == 0 && !full(k_full, t + 1)) break;
                            scores(qt, t + 1);
                            if (qt == 1) tc_commit(one, k_empty + 8 * ((t + 1) & 1));
                        }
                    }
                }
            } else {
                for (int t = 0; t < 2 && t < tiles_n; ++t)
                    if (full(k_full, t)) {
                        scores(0, t);
                        tc_commit(one, k_empty + 8 * t);
                    }
                for (int t = 0; ok && t < tiles_n; ++t) {
                    if (!full(v_full, t) || !full(p_full, t)) break;
                    values(0, t);
                    tc_commit(one, v_empty + 8 * (t & 1));
                    tc_commit(one, o_done);
                    if (t + 2 < tiles_n) {
                        if (!full(k_full, t + 2)) break;
                        scores(0, t + 2);
                        tc_commit(one, k_empty + 8 * (t & 1));
                    }
                }
            }
            tc_commit(one, done);
        }
        __syncwarp();
    } else {
        // ── tiles ──
        if constexpr (DIRECT) {
            convert_tiles<D>(r, b, h, t_begin, tiles_n, kv_end, warp - C::LOAD, k_at, v_at, k_full, k_empty, v_full, v_empty, s_fac,
                             f_full, &s_failed);
        } else if (lane == 0) {
            const uint8_t* from = kv_tiles + ((int64_t)slot * tiles_max + t_begin) * (2 * C::KV_TILE);
            const float4* fac = factors + ((int64_t)slot * tiles_max + t_begin) * C::BPT;
            int nk = 0, nv = 0;   // copies begun
            for (int t = 0; t < tiles_n; ++t, from += 2 * C::KV_TILE) {
                const int buf = t & 1, par = ((t >> 1) & 1) ^ 1;   // the first pass over the two buffers does not wait
                if (t >= 2 && !mbar_wait(k_empty + 8 * buf, par, &s_failed)) break;
                // The factors' ring of four: a K buffer is free again when both row tiles' softmax is three tiles
                // back, so the factors of four tiles back have been used.
                bulk_load(smem_u32(s_fac[t & 3]), fac + t * C::BPT, C::BPT * 16, f_full + 8 * (t & 3));
                bulk_load(k_at + buf * C::KV_TILE, from, C::KV_TILE, k_full + 8 * buf);
                ++nk;
                if (t >= 2 && !mbar_wait(v_empty + 8 * buf, par, &s_failed)) break;
                bulk_load(v_at + buf * C::KV_TILE, from + C::KV_TILE, C::KV_TILE, v_full + 8 * buf);
                ++nv;
            }
            // no copy is in flight when the CTA ends, whatever became of the other warps
            for (int i = nk - 2; i < nk; ++i)
                if (i >= 0) mbar_wait_issued(k_full + 8 * (i & 1), (i >> 1) & 1);
            for (int i = nk - 4; i < nk; ++i)
                if (i >= 0) mbar_wait_issued(f_full + 8 * (i & 3), (i >> 2) & 1);
            for (int i = nv - 2; i < nv; ++i)
                if (i >= 0) mbar_wait_issued(v_full + 8 * (i & 1), (i >> 1) & 1);
        }
        __syncwarp();
    }

    // ── the output rows: O / l through shared memory (the tiles are free once all products are done, which is waited
    // for after a failed wait, too: the products that were issued before it still read the tiles and write TMEM) ──
    if (tiles_n > 0 && !mbar_wait_issued(done, 0)) s_failed = 1;
    tc_fence_after();
    __syncthreads();
    const bool fine = s_failed == 0;
    float* rows = reinterpret_cast<float*>(tiles);
    // chunk c (4 floats) of a row at c ^ (row & 7)
    if (warp < C::SOFT_WARPS) {
        const int qt = warp / (4 * TPR), half = TPR == 2 ? (warp >> 2) & 1 : 0, row = qt * 128 + (warp & 3) * 32 + lane;
        const uint32_t o_at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + o_col + qt * 128;
        // a failed wait's rows are NaN, and the log-sum-exp of a split's is +inf, which makes NaN of what the merge joins
        // with it: nothing that a caller could take for an answer
        if (!fine && half == 0) s_lse[row] = splits > 1 ? INFINITY : NAN;
        const float inv = s_f[row];
#pragma unroll 1
        for (int c = half * (D / TPR / 32); c < (half + 1) * (D / TPR / 32); ++c) {
            uint32_t x[32];
            if (tiles_n > 0 && fine) {
                tc_ld32(o_at + 32 * c, x);
                tc_wait_ld(x);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = 0;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float4 y = make_float4(__uint_as_float(x[4 * j]) * inv, __uint_as_float(x[4 * j + 1]) * inv,
                                       __uint_as_float(x[4 * j + 2]) * inv, __uint_as_float(x[4 * j + 3]) * inv);
                if (inv == 0.0f) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (!fine) y = make_float4(NAN, NAN, NAN, NAN);
                reinterpret_cast<float4*>(rows + row * D)[(8 * c + j) ^ (row & 7)] = y;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == C::ISSUE) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
    if (!fine && threadIdx.x == 0 && r.status) atomicMax(r.status, (int)TQ_ERROR_TIMEOUT);
    for (int base = warp * (32 / LPR); base < ROWS; base += C::WARPS * (32 / LPR)) {
        const int row = base + lane / LPR, e0 = (lane % LPR) * 16, gr = row0 + row, i = gr / r.grp;
        float v[16];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4 x = reinterpret_cast<const float4*>(rows + row * D)[(e0 / 4 + c) ^ (row & 7)];
            v[4 * c] = x.x; v[4 * c + 1] = x.y; v[4 * c + 2] = x.z; v[4 * c + 3] = x.w;
        }
        if (splits > 1) {
            const int64_t at = (unit * splits + split) * ROWS + row;
            put16<float>(part, at * D + e0, v);
            if (e0 == 0) part_lse[at] = s_lse[row];
            continue;
        }
        if (r.v_rotated) fwht16<D>(v, r.norm);
        if (gr < total_rows) {
            const int hq = h * r.grp + gr % r.grp;
            store_row16(r.out_dtype, r.out, b * r.os[0] + hq * r.os[1] + (int64_t)i * r.os[2] + e0, v);
            if (r.lse && e0 == 0) r.lse[((int64_t)b * r.Hq + hq) * r.n + i] = s_lse[row];
        }
    }
}

// Work memory: partial sums of split units, then tiles and factors, each of one pass's pairs.  A pass begins when the
// one before has ended (its first kernel is launched in stream order), so they share it.
template <int D, int QTILES, bool LO, bool TREE>
static cudaError_t launch_prompt_d(const Q8Run& r, const Q8Plan& p, float* part, float* part_lse, uint8_t* tiles, cudaStream_t st) {
    using C = PromptCfg<D, false, QTILES>;
    cudaError_t e = allow_smem(attn_q8_prompt_kernel<D, false, QTILES, LO, TREE>, C::SMEM);
    if (e != cudaSuccess) return e;
    float4* factors = reinterpret_cast<float4*>(tiles + (size_t)p.pairs_pass * p.tiles_max * (2 * C::KV_TILE));
    const int64_t pairs = (int64_t)r.B * r.Hkv;
    for (int64_t pair0 = 0; pair0 < pairs; pair0 += p.pairs_pass) {
        const int now = (int)(pairs - pair0 < p.pairs_pass ? pairs - pair0 : p.pairs_pass);
        const int64_t grid = (int64_t)now * p.row_tiles * p.splits, expand = (int64_t)now * p.tiles_max;
        if (grid >= (int64_t(1) << 31) || expand >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
        expand_q8_kernel<D><<<(unsigned)expand, 256, 0, st>>>(r, pair0, p.tiles_max, tiles, factors);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3(C::WARPS * 32);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, attn_q8_prompt_kernel<D, false, QTILES, LO, TREE>, r, pair0, now, p.tiles_max, (const uint8_t*)tiles,
                               (const float4*)factors, p.row_tiles, p.splits, part, part_lse);
        if (e == cudaSuccess && p.splits > 1) e = launch_q8_merge(r, p, pair0, now, part, part_lse, st);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <int D, bool LO, bool TREE>
static cudaError_t launch_direct_d(const Q8Run& r, const Q8Plan& p, float* part, float* part_lse, cudaStream_t st) {
    using C = PromptCfg<D, true, 1>;
    cudaError_t e = allow_smem(attn_q8_prompt_kernel<D, true, 1, LO, TREE>, C::SMEM);
    if (e != cudaSuccess) return e;
    const int64_t pairs = (int64_t)r.B * r.Hkv, grid = pairs * p.row_tiles * p.splits;
    if (grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    attn_q8_prompt_kernel<D, true, 1, LO, TREE><<<(unsigned)grid, C::WARPS * 32, C::SMEM, st>>>(r, 0, (int)pairs, 0, nullptr, nullptr, p.row_tiles,
                                                                                   p.splits, part, part_lse);
    e = cudaGetLastError();
    return e == cudaSuccess && p.splits > 1 ? launch_q8_merge(r, p, 0, (int)pairs, part, part_lse, st) : e;
}

cudaError_t launch_attention_q8_prompt(const Q8Run& r, const Q8Plan& p, float* part, float* part_lse, void* tiles, cudaStream_t st) {
    uint8_t* t = static_cast<uint8_t*>(tiles);
    const auto run = [&](auto lo, auto tree) {
        constexpr bool LO = decltype(lo)::value, TREE = decltype(tree)::value;
        if (p.direct) return r.D == 256 ? launch_direct_d<256, LO, TREE>(r, p, part, part_lse, st) : launch_direct_d<128, LO, TREE>(r, p, part, part_lse, st);
        if (!LO && p.rows == 256) return launch_prompt_d<128, 2, false, TREE>(r, p, part, part_lse, t, st);
        return r.D == 256 ? launch_prompt_d<256, 1, LO, TREE>(r, p, part, part_lse, t, st) : launch_prompt_d<128, 1, LO, TREE>(r, p, part, part_lse, t, st);
    };
    const std::true_type yes;
    const std::false_type no;
    if (r.tree) return p.lo ? run(yes, yes) : run(no, yes);
    return p.lo ? run(yes, no) : run(no, no);
}

// Query rows of a CTA.  Two row tiles of D = 128 hide each other's softmax and products (8192-token prompt 597 us, with
// one 734 us), where there are enough of them: under half of the SMs, more and smaller CTAs end sooner (256 tokens of 32
// heads 15 us, with two 22 us; 512: 18 and 26 us; from 80 CTAs of two on two are faster: 300 tokens of two sequences
// behind 4000 103 and 115 us, 1024 tokens 35 and 37 us).  With q' as two terms there is no room for a second one in TMEM
// (with 64 tokens at a time there is: 783 us for the 8192-token prompt, with one row tile 750 us).
int q8_prompt_rows(int64_t pairs, int64_t rows, int D, bool direct, bool lo) {
    return D == 128 && !direct && !lo && 2 * pairs * ((rows + 255) / 256) >= sm_count() ? 256 : 128;
}

// tiles of one pass: all pairs, or as many as 1 GiB holds
void q8_prompt_tiles(int64_t pairs, int D, int64_t max_len, Q8Plan* p) {
    const int kt = D == 128 ? PromptCfg<128, false, 1>::KT : PromptCfg<256, false, 1>::KT;
    p->tiles_max = (int)((max_len + kt - 1) / kt);
    const int64_t bytes = (int64_t)p->tiles_max * (4 * kt * D + kt);   // two f16 tiles, 16 bytes per 16 tokens
    const int64_t most = bytes > 0 ? (int64_t(1) << 30) / bytes : pairs;
    p->pairs_pass = (int)(most < 1 ? 1 : (most < pairs ? most : pairs));
    p->tile_bytes = (size_t)bytes * p->pairs_pass;
}

}  // namespace tq
