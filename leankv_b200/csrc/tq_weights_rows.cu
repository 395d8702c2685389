// tq_weights_rows.cu — sums of attention weights over 8-bit keys for many query rows (prompts, windows of them), on tcgen05.
//
// The mathematics is tq_weights.cu's.  With many rows per KV head the products and the exponentials bound it, not the keys.
// Scores are computed as K Q^T, tokens on the lanes of TMEM and query rows on its columns: a thread then adds up the weights of
// its token over the columns that it reads, with nothing to exchange but the sums of four threads at the end, and tokens' sums
// leave the kernel as one float.
//
// Products are of 8-bit whole numbers with 32-bit sums (kind::i8): codes enter as they lie in the pages.  A row of q' is the sum
// of three terms of 8 bits, q1 + q2 / 128 + q3 / 128^2, in units of 1/127 of its largest element; the terms are rows of the same
// product, N = 3 x 64.  Two f16 terms take as many operations, but the codes have to be converted on their way and the
// fp32 sums were off by 4e-6 of the result, where this is off by 1e-6: sums of whole numbers are exact.
//
// What bounds it: the way from TMEM to the weights, 13 instructions issued for each of them, half of them its arithmetic, and their
// latency: no pipe is full.  The last 64 tokens of 32 heads over 2 x 16100 tokens (256 rows a KV head): 56 us with the preparing
// kernel, floor 10 (this kernel alone: issue 55 %, FMA pipe 41 %, special function unit 33 %, tensor pipe 25 %, 20 warps an SM); with
// f16 products 38 us, with mma.sync 210.  Terms joined by a shift, which rounds down, took 53 us and made all scores too small.
// One scale for 64 rows: 4 us less, but rows much smaller than their neighbours lost bits.  Four converting warps more, deeper rings, sums
// begun from the bits of 1.5 * 2^23 in TMEM (61 to 88 us): slower.
//
// weights_rows_prepare_kernel: q' (Hadamard, the row's scale, terms) into images of the shared-memory tiles, once per call (a row is
// read by every CTA of its KV head); with each row's scale, log-sum-exp and last token.
//
// weights_rows_kernel: a CTA takes a run of tokens of one (sequence, KV head) and QN rows at a time, whose images stay in shared
// memory while the run's keys come by, 128 tokens at a time.  Warps:
//   3      copy codes (cp.async, 16 bytes a lane, in the products' 128-byte swizzle)
//   1      issues the products: 128 tokens x 64 rows x 3 terms, two buffers in TMEM
//   2 x 8  take turns at the 64 rows' scores, two threads a token: terms from TMEM, weights, sums
// A token's sums stay in shared memory, one for each of its four threads, until all rows have been taken, QN at a time.  Tiles of which no row sees a token
// (prompts' later halves) are left out.
//
// Every wait gives up after about a second (TQ_ERROR_TIMEOUT; the run's weights become NaN) instead of hanging; copies and
// products that were issued before are waited for.
#include <type_traits>

#include "leankv_tq.h"
#include "tq_attn_q8.cuh"
#include "tq_evict.h"
#include "tq_kernels.h"
#include "tq_tc.cuh"
#include "tq_warp_rows.cuh"

namespace tq {

constexpr int WR_SUB = 64, WR_N = 3 * WR_SUB;   // rows of a product, and its columns

template <int D> struct WrCfg {
    static constexpr int NS = D == 128 ? 4 : 2, QN = WR_SUB * NS;              // products of a tile of keys, rows at a time
    static constexpr int SEGS = D / 128, STAGES = D == 128 ? 4 : 3;            // runs of 128 bytes of a row; tiles of keys under way
    static constexpr int QSEG = WR_N * 128, QSUB = SEGS * QSEG, QTILE = NS * QSUB;   // bytes
    static constexpr int KSEG = 128 * 128, KTILE = SEGS * KSEG;
    static constexpr int EPI = 16, ISSUE = EPI, COPY = EPI + 1, COPY_WARPS = 3, WARPS = COPY + COPY_WARPS, THREADS = 32 * WARPS;
    static constexpr int TOKENS = 2048;                                        // of a CTA whose sums are kept at a time
    static constexpr int SMEM = 1024 + QTILE + STAGES * KTILE + 4 * TOKENS * 4;
};

// Whole numbers below 2^22 in size plus the bits of 1.5 * 2^23 are floats of that and themselves: conversions by instruction would
// take as much of the special function unit as the powers do.
constexpr uint32_t WR_ZERO = 0x4B400000u;

struct RowMeta {
    float nl;      // negative log-sum-exp, in the log2 domain
    float f;       // of its scores, into that domain
    int lim;       // last token that the row sees, -1: none
};

__device__ __forceinline__ void wr_mma(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
// s8 operands, s32 sums, M = 128, N = 192, both with K contiguous
constexpr uint32_t WR_IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(WR_N >> 3) << 17) | (8u << 24);
// 8 columns of each of the three terms of this thread's TMEM lane
__device__ __forceinline__ void wr_load(uint32_t a, uint32_t (&x)[3][8]) {
#pragma unroll
    for (int k = 0; k < 3; ++k)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(x[k][0]), "=r"(x[k][1]), "=r"(x[k][2]), "=r"(x[k][3]), "=r"(x[k][4]), "=r"(x[k][5]), "=r"(x[k][6]), "=r"(x[k][7])
                     : "r"(a + k * WR_SUB));
}
// what was loaded is there; tied to it, so that nothing that uses it can be moved before
__device__ __forceinline__ void wr_wait(uint32_t (&x)[3][8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0][0]), "+r"(x[0][1]), "+r"(x[0][2]), "+r"(x[0][3]), "+r"(x[0][4]), "+r"(x[0][5]), "+r"(x[0][6]), "+r"(x[0][7]) :: "memory");
#pragma unroll
    for (int k = 1; k < 3; ++k)
        asm volatile("" : "+r"(x[k][0]), "+r"(x[k][1]), "+r"(x[k][2]), "+r"(x[k][3]), "+r"(x[k][4]), "+r"(x[k][5]), "+r"(x[k][6]), "+r"(x[k][7]));
}

// One CTA: 64 rows of a (sequence, KV head), 8 a warp.
template <int D>
__global__ void __launch_bounds__(256) weights_rows_prepare_kernel(const WeightsRun p, int64_t pair0, int subs, uint8_t* __restrict__ images,
                                                                   RowMeta* __restrict__ meta) {
    using C = WrCfg<D>;
    constexpr int E = D / 32, ROWS = WR_SUB / 8;
    const Q8Run& r = p.q;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t slot = blockIdx.x / subs, pair = pair0 + slot;
    const int sub = blockIdx.x % subs, h = (int)(pair % r.Hkv), b = (int)(pair / r.Hkv);
    const SeqLens sl = seq_lens(r, b);
    const int i0 = sl.q_len > p.window ? sl.q_len - (int)p.window : 0;
    // Row k's log-sum-exp, -inf for a row that sees no token, whatever was left for it.  Such a row, and one of -inf, adds nothing,
    // whatever q holds there.
    const auto lse_of = [&](int i, int hq) { return last_seen(r, sl, i) >= 0 ? p.lse[((int64_t)b * r.Hq + hq) * r.n + i] : -INFINITY; };
    float v[ROWS][E], inv[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const int at = sub * WR_SUB + warp * ROWS + k, i = i0 + at / r.grp, hq = h * r.grp + at % r.grp;
#pragma unroll
        for (int j = 0; j < E; ++j) v[k][j] = 0.0f;
        if (lse_of(i, hq) != -INFINITY) load_some<E>(r.q_dtype, r.q, b * r.qs[0] + hq * r.qs[1] + (int64_t)i * r.qs[2] + lane * E, v[k]);
    }
    float mine = 0.0f;   // lane k < ROWS: the largest element of row k
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        if (r.rotate_q) fwht_warp<E>(v[k], r.norm);
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) top = fmaxf(top, fabsf(v[k][j]));
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));   // floats from 0 on are in the order of their bits
        if (lane == k) mine = top;
        inv[k] = top >= 0x1p-100f ? __fdiv_rn(127.0f, top) : 0.0f;
    }
    uint8_t* image = images + (slot * subs + sub) * C::QSUB;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const int row = warp * ROWS + k, e0 = lane * E, c = (e0 & 127) >> 4;
        uint32_t q[3][E / 4];
#pragma unroll
        for (int j = 0; j < E / 4; ++j) {
            q[0][j] = q[1][j] = q[2][j] = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float y = v[k][4 * j + x] * inv[k], a = rintf(y), z = (y - a) * 128.0f, d = rintf(z), f = rintf((z - d) * 128.0f);
                q[0][j] |= ((uint32_t)(int)a & 0xFFu) << (8 * x);
                q[1][j] |= ((uint32_t)(int)d & 0xFFu) << (8 * x);
                q[2][j] |= ((uint32_t)(int)f & 0xFFu) << (8 * x);
            }
        }
#pragma unroll
        for (int term = 0; term < 3; ++term) {
            const int n = term * WR_SUB + row;
            uint8_t* to = image + (e0 >> 7) * C::QSEG + n * 128 + ((c ^ (n & 7)) << 4) + (e0 & 15);
#pragma unroll
            for (int j = 0; j < E / 4; ++j) reinterpret_cast<uint32_t*>(to)[j] = q[term][j];
        }
    }
    if (lane < ROWS) {
        const int at = sub * WR_SUB + warp * ROWS + lane, i = i0 + at / r.grp, hq = h * r.grp + at % r.grp;
        const float lse = lse_of(i, hq);
        const bool sees = lse != -INFINITY;
        RowMeta m;
        m.nl = sees ? -lse * LOG2E : -INFINITY;
        m.f = mine * (r.sm_scale * LOG2E * (1.0f / 127.0f));
        m.lim = sees ? last_seen(r, sl, i) : -1;
        meta[(slot * subs + sub) * WR_SUB + warp * ROWS + lane] = m;
    }
}

template <int D>
__global__ void __launch_bounds__(WrCfg<D>::THREADS, 1)
weights_rows_kernel(const WeightsRun p, int64_t pair0, int splits, int subs, const uint8_t* __restrict__ images, const RowMeta* __restrict__ meta) {
    using C = WrCfg<D>;
    constexpr int QN = C::QN, NS = C::NS, STAGES = C::STAGES;
    const Q8Run& r = p.q;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[16];
    __shared__ __align__(16) float s_row[2 * QN];   // of two rows: their nl, their f
    __shared__ int s_lim[QN], s_most, s_least;   // last tokens of the rows; the largest and the least of them
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    uint8_t* tiles_at = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t q_at = smem_u32(tiles_at), k_at = q_at + C::QTILE, bar0 = smem_u32(bars);
    float* s_sum = reinterpret_cast<float*>(tiles_at + C::QTILE + STAGES * C::KTILE);   // [thread of a token][token]
    const uint32_t k_full = bar0, k_empty = bar0 + 32, s_full = bar0 + 64, s_empty = bar0 + 80, q_full = bar0 + 96, done = bar0 + 104;

    const int split = blockIdx.x % splits, slot = blockIdx.x / splits;
    const int64_t pair = pair0 + slot;
    const int h = (int)(pair % r.Hkv), b = (int)(pair / r.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const SeqLens sl = seq_lens(r, b);
    const int per = ((sl.len + splits - 1) / splits + 127) & ~127;
    const int64_t begin64 = (int64_t)split * per;
    if (begin64 >= sl.len) {
        asm volatile("griddepcontrol.wait;" ::: "memory");   // this grid does not end before the images' kernel
        return;
    }
    const int begin_all = (int)begin64, end_all = sl.len - begin_all < per ? sl.len : begin_all + per;
    const int fresh = p.fresh ? p.fresh[b] : 0x7fffffff;
    const int rows = (int)(sl.q_len > p.window ? p.window : sl.q_len) * r.grp, chunks = rows ? (rows + QN - 1) / QN : 1;
    const int32_t* pages = r.pages + (int64_t)b * r.max_pages;
    const int per_page = r.page_shift - 4;
    auto block_in = [&](int page, int block) {   // of the pool, -1 for a page outside it
        return page < 0 || page >= r.num_pages ? -1 : (int)((((int64_t)page * r.Hkv + h) << per_page) + (block & ((1 << per_page) - 1)));
    };

    if (threadIdx.x == 0) {
        s_failed = 0;
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(k_full + 8 * i, C::COPY_WARPS);
            mbar_init(k_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(s_empty + 8 * i, C::EPI / 2);
        }
        mbar_init(q_full, 1);
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C::ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the images are there
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);

    // alike in all warps: tiles of keys so far, products (of 64 rows) so far, chunks of rows so far
    int seq = 0, prod = 0, loads = 0;
    bool fail = false;
    for (int begin = begin_all; begin < end_all; begin += C::TOKENS) {
    const int end = end_all - begin < C::TOKENS ? end_all : begin + C::TOKENS, all = (end - begin + 127) >> 7;
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const int left_rows = rows - chunk * QN, ns = left_rows >= QN ? NS : (left_rows + WR_SUB - 1) / WR_SUB;   // 0 without rows
        const int64_t sub0 = (int64_t)slot * subs + chunk * NS;
        // the rows before are no longer used (their products have been waited for); all leave together after a failed wait
        fail = __syncthreads_or(s_failed) != 0;
        if (fail) break;
        if (threadIdx.x == 0 && ns > 0) {
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(q_full), "r"(ns * C::QSUB) : "memory");
            for (int i = 0; i < ns; ++i)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(q_at + i * C::QSUB), "l"(images + (sub0 + i) * C::QSUB), "r"(C::QSUB), "r"(q_full) : "memory");
        }
        if (threadIdx.x == 0) {
            s_most = -1;
            s_least = 0x7fffffff;
        }
        __syncthreads();
        if (threadIdx.x < ns * WR_SUB) {
            const RowMeta m = meta[sub0 * WR_SUB + threadIdx.x];
            s_row[(threadIdx.x >> 1) * 4 + (threadIdx.x & 1)] = m.nl;
            s_row[(threadIdx.x >> 1) * 4 + 2 + (threadIdx.x & 1)] = m.f;
            s_lim[threadIdx.x] = m.lim;
            const int most = __reduce_max_sync(0xffffffffu, m.lim), least = __reduce_min_sync(0xffffffffu, m.lim < 0 ? 0x7fffffff : m.lim);
            if (lane == 0) {
                atomicMax(&s_most, most);
                atomicMin(&s_least, least);
            }
        }
        __syncthreads();
        // tiles of keys that some row sees
        const int most = s_most, least = s_least, act = most < begin ? 0 : min(all, ((most - begin) >> 7) + 1);

        if (warp < C::EPI) {
            // ── weights and sums: thread = token and 32 of the rows of every other product ──
            const int odd = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane, part = odd * 2 + half;
            const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16) + odd * 256 + half * 32;
            // the token's scale a tile ahead, and its page two (what is loaded is not looked at before its turn: the warp would wait)
            int next_page = -1;
            float next_ks = 0.0f;
            auto locate = [&](int t) {
                const int tok = begin + t * 128 + row;
                next_page = -1;
                if (t < all && tok < end) next_page = pages[tok >> r.page_shift];
            };
            auto fetch = [&](int t) {
                const int tok = begin + t * 128 + row;
                const int blk = block_in(next_page, tok >> 4);
                next_ks = blk >= 0 ? r.ks[blk] : 0.0f;
            };
            locate(0);
            fetch(0);
            locate(1);
            bool ok = true;
            for (int t = 0; t < all; ++t) {
                const int tok0 = begin + t * 128, tok = tok0 + row;
                const float2 ks = make_float2(next_ks, next_ks);
                fetch(t + 1);
                locate(t + 2);
                float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
                if (t < act) {
                    const bool edge = tok0 + 127 > least;
                    const int first = prod + t * ns;             // of the tile's products
#pragma unroll
                    for (int i = 0; i < (NS + 1) / 2; ++i) {
                        const int j = ((first + odd) & 1) + 2 * i, n = first + j;
                        if (j >= ns) continue;
                        ok = ok && __all_sync(0xffffffffu, mbar_wait(s_full + 8 * odd, (n >> 1) & 1, &s_failed));
                        if (!ok) continue;
                        tc_fence_after();
                        uint32_t raw[2][3][8];   // 8 rows' terms are loaded while those before are used
                        wr_load(from, raw[0]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t(&x)[3][8] = raw[c & 1];
                            wr_wait(x);
                            if (c < 3) wr_load(from + 8 * (c + 1), raw[(c + 1) & 1]);
                            const int r0 = j * WR_SUB + half * 32 + 8 * c;
                            float e[8];
#pragma unroll
                            for (int k = 0; k < 8; k += 4) {
                                const float4 l = *reinterpret_cast<const float4*>(s_row + 2 * (r0 + k)), m = *reinterpret_cast<const float4*>(s_row + 2 * (r0 + k) + 4);
                                // c1 + (c2 + c3 / 128) / 128, floats from the bits of 1.5 * 2^23 + c.  c2 + c3 / 128 is rounded to a
                                // whole number there, the nearest, so that scores are off by up to half of 1/128 of c1's unit, either way.
                                const float2 off = make_float2(-12681984.0f, -12681984.0f), m1 = make_float2(0x1p-7f, 0x1p-7f);
                                const auto term = [&](int t, int u) {
                                    return make_float2(__uint_as_float(x[t][k + u] + WR_ZERO), __uint_as_float(x[t][k + u + 1] + WR_ZERO));
                                };
                                const auto sum = [&](int u) {
                                    return __ffma2_rn(__ffma2_rn(term(2, u), m1, term(1, u)), m1, __fadd2_rn(term(0, u), off));
                                };
                                const float2 y = __ffma2_rn(sum(0), __fmul2_rn(make_float2(l.z, l.w), ks), make_float2(l.x, l.y));
                                const float2 z = __ffma2_rn(sum(2), __fmul2_rn(make_float2(m.z, m.w), ks), make_float2(m.x, m.y));
                                e[k] = ex2(y.x);
                                e[k + 1] = ex2(y.y);
                                e[k + 2] = ex2(z.x);
                                e[k + 3] = ex2(z.y);
                            }
                            if (edge) {
                                asm volatile("" ::: "memory");   // few tiles: kept a branch
#pragma unroll
                                for (int k = 0; k < 8; ++k)
                                    if (tok > s_lim[r0 + k]) e[k] = 0.0f;
                            }
                            if (c == 3) {   // the buffer has been read
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(s_empty + 8 * odd);
                            }
#pragma unroll
                            for (int k = 0; k < 8; k += 4) {
                                sum0 = __fadd2_rn(sum0, make_float2(e[k], e[k + 1]));
                                sum1 = __fadd2_rn(sum1, make_float2(e[k + 2], e[k + 3]));
                            }
                        }
                    }
                }
                float* at = s_sum + part * C::TOKENS + t * 128 + row;
                const float x = (sum0.x + sum0.y) + (sum1.x + sum1.y);
                *at = chunk > 0 ? *at + x : x;
            }
        } else if (warp == C::ISSUE) {
            // ── products ──
            if (ns > 0) {
                const uint32_t one = tc_elect();
                const uint64_t k_desc = tile_desc(k_at, 16), q_desc = tile_desc(q_at, 16);
                bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, loads & 1, &s_failed));
                for (int t = 0; ok && t < act; ++t) {
                    const int stage = (seq + t) % STAGES;
                    ok = __all_sync(0xffffffffu, mbar_wait(k_full + 8 * stage, ((seq + t) / STAGES) & 1, &s_failed));
                    for (int j = 0; ok && j < ns; ++j) {
                        const int n = prod + t * ns + j, buf = n & 1;
                        if (n >= 2) ok = __all_sync(0xffffffffu, mbar_wait(s_empty + 8 * buf, ((n >> 1) & 1) ^ 1, &s_failed));
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t k = k_desc + stage * (C::KTILE >> 4), q = q_desc + j * (C::QSUB >> 4);
#pragma unroll
                        for (int s = 0; s < D / 32; ++s)
                            wr_mma(one, tmem + buf * 256, k + ((s >> 2) * (C::KSEG >> 4) + (s & 3) * 2),
                                   q + ((s >> 2) * (C::QSEG >> 4) + (s & 3) * 2), WR_IDESC, s > 0);
                        tc_commit(one, s_full + 8 * buf);
                    }
                    if (ok) tc_commit(one, k_empty + 8 * stage);
                }
            }
            __syncwarp();
        } else {
            // ── codes: a warp takes every third block of 16 tokens; STAGES - 1 tiles are under way ──
            const int cw = warp - C::COPY;
            int page = -1;   // lanes 0 .. 7: of the tile's blocks
            auto locate = [&](int t) {
                const int tok = begin + t * 128 + lane * 16;
                page = -1;
                if (lane < 8 && t < act && tok < end) page = pages[tok >> r.page_shift];
            };
            auto landed = [&](int t) {   // tile t's copies of this warp: for the products to read
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full + 8 * ((seq + t) % STAGES));
            };
            locate(0);
            bool ok = true;
            for (int t = 0; ok && t < act; ++t) {
                const int n = seq + t, stage = n % STAGES;
                if (n >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(k_empty + 8 * stage, ((n / STAGES) & 1) ^ 1, &s_failed));
                if (ok) {
                    const int blk = block_in(page, (begin + t * 128 + lane * 16) >> 4);
                    for (int block = cw; block < 8; block += C::COPY_WARPS) {
                        const int at = __shfl_sync(0xffffffffu, blk, block);
                        if (at < 0) continue;   // whatever lies there: its tokens' sums are not kept
                        const int8_t* src = r.k + (int64_t)at * (16 * D) + lane * 16;
#pragma unroll
                        for (int e = 0; e < D / 32; ++e) {
                            const int c = lane + 32 * e, x = block * 16 + c / (D / 16), cc = c % (D / 16);
                            const uint32_t to = k_at + stage * C::KTILE + (cc >> 3) * C::KSEG + x * 128 + (((cc & 7) ^ (x & 7)) << 4);
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src + e * 512) : "memory");
                        }
                    }
                    locate(t + 1);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
                if (ok && t >= STAGES - 1) landed(t - (STAGES - 1));
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (ok)
                for (int t = act > STAGES - 1 ? act - (STAGES - 1) : 0; t < act; ++t) landed(t);
        }
        seq += act;
        prod += act * ns;
        if (ns > 0) ++loads;
    }
    if (fail) break;
    __syncthreads();
    for (int tok = begin + threadIdx.x; tok < end; tok += C::THREADS) {   // a token's four sums
        const int blk = block_at(r, b, h, tok >> 4);
        if (blk < 0) {
            if (r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
            continue;
        }
        const float* sums = s_sum + (tok - begin);
        const float x = (sums[0] + sums[C::TOKENS]) + (sums[2 * C::TOKENS] + sums[3 * C::TOKENS]);
        float* at = p.weights + (int64_t)blk * 16 + (tok & 15);
        *at = tok < fresh && p.decay != 0.0f ? fmaf(p.decay, *at, x) : x;
    }
    }

    // copies and products that were issued end before the memory is given back
    if (warp == C::ISSUE) {
        const uint32_t one = tc_elect();
        tc_commit(one, done);
        __syncwarp();
    }
    if (loads > 0) mbar_wait_issued(q_full, (loads - 1) & 1);
    if (!mbar_wait_issued(done, 0)) s_failed = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == C::ISSUE) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
    if (s_failed) {
        if (threadIdx.x == 0 && r.status) atomicMax(r.status, (int)TQ_ERROR_TIMEOUT);
        for (int tok = begin_all + threadIdx.x; tok < end_all; tok += C::THREADS) {
            const int blk = block_at(r, b, h, tok >> 4);
            if (blk >= 0) p.weights[(int64_t)blk * 16 + (tok & 15)] = NAN;
        }
    }
}

// bytes of the work memory for a product's rows: image, meta
template <int D> constexpr size_t wr_sub_bytes() { return WrCfg<D>::QSUB + WR_SUB * sizeof(RowMeta); }

// A CTA's time is its tokens for each chunk of rows plus a start for each; one CTA an SM.  Its tokens at most fill the sums'
// place once where there are several chunks (beyond, it would read the rows again).
void weights_rows_plan(int64_t pairs, int D, int64_t rows, int64_t len, WeightsPlan* p) {
    const int qn = D == 128 ? WrCfg<128>::QN : WrCfg<256>::QN, sums = WrCfg<128>::TOKENS;
    p->rows = qn;
    p->chunks = (int)((rows + qn - 1) / qn);
    p->tiles = (int)((rows + WR_SUB - 1) / WR_SUB);
    const int64_t each = (int64_t)(D == 128 ? wr_sub_bytes<128>() : wr_sub_bytes<256>()) * p->tiles, most = int64_t(1) << 30;
    const int64_t pass = most / each;
    p->pairs_pass = (int)(pass < 1 ? 1 : (pass < pairs ? pass : pairs));
    p->bytes = (size_t)p->pairs_pass * each;
    const int64_t slots = sm_count(), start = 512;
    int64_t best = INT64_MAX;
    for (int s = 1; s <= 256; ++s) {
        const int64_t per = ((len + s - 1) / s + 127) / 128 * 128;
        if (s > 1 && (int64_t)(s - 1) * per >= len) continue;
        const int64_t waves = (p->pairs_pass * s + slots - 1) / slots, turns = (per + sums - 1) / sums;
        const int64_t cost = waves * (per + start * turns);
        if (cost < best) { best = cost; p->splits = s; }
        if (waves > 8) break;
    }
}

template <int D>
static cudaError_t launch_weights_rows_d(const WeightsRun& r, const WeightsPlan& p, uint8_t* ws, cudaStream_t st) {
    using C = WrCfg<D>;
    cudaError_t e = allow_smem(weights_rows_kernel<D>, C::SMEM);
    if (e != cudaSuccess) return e;
    const size_t all = (size_t)p.pairs_pass * p.tiles;
    RowMeta* meta = reinterpret_cast<RowMeta*>(ws + all * C::QSUB);
    const int64_t pairs = (int64_t)r.q.B * r.q.Hkv;
    for (int64_t pair0 = 0; pair0 < pairs; pair0 += p.pairs_pass) {
        const int now = (int)(pairs - pair0 < p.pairs_pass ? pairs - pair0 : p.pairs_pass);
        const int64_t prepare = (int64_t)now * p.tiles, grid = (int64_t)now * p.splits;
        if (prepare >= (int64_t(1) << 31) || grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
        weights_rows_prepare_kernel<D><<<(unsigned)prepare, 256, 0, st>>>(r, pair0, p.tiles, ws, meta);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3(C::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, weights_rows_kernel<D>, r, pair0, p.splits, p.tiles, (const uint8_t*)ws, (const RowMeta*)meta);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_weights_rows(const WeightsRun& r, const WeightsPlan& p, void* workspace, cudaStream_t st) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    return r.q.D == 256 ? launch_weights_rows_d<256>(r, p, ws, st) : launch_weights_rows_d<128>(r, p, ws, st);
}

}  // namespace tq
