// tq_weights_rows.cu — sums of attention weights over 8-bit keys for many query rows (prompts, windows of them), on tcgen05.
//
// The mathematics is tq_weights.cu's.  With many rows per KV head the products and the exponentials bound it, not the keys.
// Scores are computed as K Q^T, tokens on the lanes of TMEM and query rows on its columns: a thread then adds up the weights of
// its token over the columns that it reads, with nothing to exchange, and tokens' sums leave the kernel as one float.
//
// weights_rows_prepare_kernel: q' (Hadamard, row maximum) as two f16 terms, into images of the shared-memory tiles, once per call
// (a row is read by every CTA of its KV head); with each row's factor, log-sum-exp and last token.
//
// weights_rows_kernel: a CTA takes a run of tokens of one (sequence, KV head) and QN rows at a time, whose images stay in shared
// memory while the run's keys come by, 128 tokens at a time.  Warps:
//   3 (7)  convert codes to f16 tiles (two buffers; in brackets: heads of 256)
//   1      issues the products: S = K (Q1 + Q2)^T, 128 tokens x QN rows, f16, fp32 sums in TMEM (two buffers)
//   2 x 8  (2 x 4) take turns at the tokens' tiles, two threads (one) a token: scores from TMEM, weights, sums
// More rows than QN are taken in turn, the run's sums kept in shared memory between.  Tiles of which no row sees a token
// (prompts' later halves) are left out.
//
// Numbers: codes are exact in f16, q' has 22 bits in two terms, sums are fp32.
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

template <int D> struct WrCfg {
    static constexpr int QN = D == 128 ? 256 : 64;                      // rows at a time
    static constexpr int TPT = D == 128 ? 2 : 1, HN = QN / TPT;          // threads that share a token, and their rows
    static constexpr int SEGS = D / 64;
    static constexpr int QTERM = QN * D * 2, QTILE = 2 * QTERM;                           // bytes
    static constexpr int KTILE = 128 * D * 2, KSEG = 128 * 128, QSEG = QN * 128;
    static constexpr int EPI = 8 * TPT, ISSUE = EPI, CONV = EPI + 1, CONV_WARPS = D == 128 ? 3 : 7, WARPS = CONV + CONV_WARPS;
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int ALL_UNITS = 8 * SEGS;                                            // of a tile: 16 tokens x 64 elements
    static constexpr int UNITS = (ALL_UNITS + CONV_WARPS - 1) / CONV_WARPS;               // of a converting warp
    static constexpr int TOKENS = 2048;                                                   // of a CTA between chunks of rows
    static constexpr int SMEM = 1024 + QTILE + 2 * KTILE + TOKENS * 4;
};

struct RowMeta {
    float f, nl;   // factor of the scores and the negative log-sum-exp, in the log2 domain
    int lim;       // last token that the row sees, -1: none
    int pad;
};

template <int D>
__global__ void __launch_bounds__(256) weights_rows_prepare_kernel(const WeightsRun p, int64_t pair0, int pairs, int tiles,
                                                                   uint8_t* __restrict__ images, RowMeta* __restrict__ meta) {
    using C = WrCfg<D>;
    constexpr int E = D / 32;
    const Q8Run& r = p.q;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 8 + warp, rows_pair = (int64_t)tiles * C::QN, slot = id / rows_pair, pair = pair0 + slot;
    const int at = (int)(id - slot * rows_pair), tile = at / C::QN, row = at % C::QN;
    if (slot >= pairs) return;
    const int h = (int)(pair % r.Hkv), b = (int)(pair / r.Hkv);
    const SeqLens sl = seq_lens(r, b);
    const int i0 = sl.q_len > p.window ? sl.q_len - (int)p.window : 0, i = i0 + at / r.grp, hq = h * r.grp + at % r.grp;
    const bool live = i < sl.q_len;
    float v[E];
    if (live) {
        load_some<E>(r.q_dtype, r.q, b * r.qs[0] + hq * r.qs[1] + (int64_t)i * r.qs[2] + lane * E, v);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = 0.0f;
    }
    const float lse = live ? p.lse[((int64_t)b * r.Hq + hq) * r.n + i] : -INFINITY;
    if (r.rotate_q) fwht_warp<E>(v, r.norm);
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
    for (int o = 1; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float inv = top >= 0x1p-100f ? __fdiv_rn(1.0f, top) : 0.0f;
    uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
        const float x = v[2 * j] * inv, y = v[2 * j + 1] * inv;
        const __half2 a = __floats2half2_rn(x, y);
        hi[j] = *reinterpret_cast<const uint32_t*>(&a);
        lo[j] = pack_h2(x - __low2float(a), y - __high2float(a));
    }
    const int e0 = lane * E, c = (e0 & 63) >> 3, sub = (e0 & 7) * 2;
    uint8_t* to = images + (slot * tiles + tile) * C::QTILE + (e0 >> 6) * C::QSEG + row * 128 + ((c ^ (row & 7)) << 4) + sub;
    if constexpr (E == 4) {
        *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(to + C::QTERM) = make_uint2(lo[0], lo[1]);
    } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(to + C::QTERM) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (lane == 0) {
        RowMeta m;
        const bool sees = lse != -INFINITY;   // a row that saw nothing adds nothing
        m.f = top * (r.sm_scale * LOG2E);
        m.nl = sees ? -lse * LOG2E : -INFINITY;
        m.lim = sees ? last_seen(r, sl, i) : -1;
        m.pad = 0;
        meta[id] = m;
    }
}

template <int D>
__global__ void __launch_bounds__(WrCfg<D>::THREADS, 1)
weights_rows_kernel(const WeightsRun p, int64_t pair0, int splits, int tiles, const uint8_t* __restrict__ images, const RowMeta* __restrict__ meta) {
    using C = WrCfg<D>;
    constexpr int QN = C::QN, HN = C::HN;
    const Q8Run& r = p.q;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[16];
    __shared__ __align__(16) float s_f[QN], s_nl[QN];
    __shared__ int s_lim[QN], s_most, s_least;   // last tokens of the rows; the largest and the least of them
    __shared__ float s_part[2][2][128];          // sums of the second half of the rows, [tile & 1][turn & 1]
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    uint8_t* tiles_at = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t q_at = smem_u32(tiles_at), k_at = q_at + C::QTILE, bar0 = smem_u32(bars);
    float* s_sum = reinterpret_cast<float*>(tiles_at + C::QTILE + 2 * C::KTILE);
    const uint32_t k_full = bar0, k_empty = bar0 + 16, s_full = bar0 + 32, s_empty = bar0 + 48, q_full = bar0 + 64, done = bar0 + 72;

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

    if (threadIdx.x == 0) {
        s_failed = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, C::CONV_WARPS);
            mbar_init(k_empty + 8 * i, 1);
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

    int seq = 0, loads = 0;   // tiles of keys whose scores have been computed, chunks of rows so far; alike in all warps
    bool fail = false;
    const int step = chunks > 1 ? C::TOKENS : per;   // sums wait for the next chunk only
    for (int begin = begin_all; begin < end_all; begin += step) {
    const int end = end_all - begin < step ? end_all : begin + step, all = (end - begin + 127) >> 7;
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const bool last = chunk + 1 == chunks;
        const int64_t tile = (int64_t)slot * tiles + chunk;
        // the rows before are no longer used (their products have been waited for); all leave together after a failed wait
        fail = __syncthreads_or(s_failed) != 0;
        if (fail) break;
        if (threadIdx.x == 0 && rows > 0) {
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(q_full), "r"(C::QTILE) : "memory");
            for (int i = 0; i < C::QTILE / 32768; ++i)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(q_at + i * 32768), "l"(images + tile * C::QTILE + i * 32768), "r"(32768), "r"(q_full) : "memory");
        }
        if (threadIdx.x == 0) {
            s_most = -1;
            s_least = 0x7fffffff;
        }
        __syncthreads();
        if (threadIdx.x < QN && rows > 0) {
            const RowMeta m = meta[tile * QN + threadIdx.x];
            s_f[threadIdx.x] = m.f;
            s_nl[threadIdx.x] = m.nl;
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
            // ── weights and sums: thread = token and half of the rows; the warps take turns at the tiles ──
            const int odd = warp / (4 * C::TPT), half = C::TPT == 2 ? (warp >> 2) & 1 : 0, row = (warp & 3) * 32 + lane;
            const int first = (seq + odd) & 1;       // of this warp's tiles: those whose scores lie in buffer `odd`
            const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16) + odd * QN + half * HN;
            // the token's block, its scale and the earlier weight, a tile ahead
            int next_blk = -1;
            float next_ks = 0.0f, next_held = 0.0f;
            auto fetch = [&](int t) {
                const int tok = begin + t * 128 + row;
                next_blk = t < all && tok < end ? block_at(r, b, h, tok >> 4) : -1;
                next_ks = next_blk >= 0 ? r.ks[next_blk] : 0.0f;
                next_held = 0.0f;
                if (next_blk >= 0 && half == 0 && last && tok < fresh && p.decay != 0.0f) next_held = p.weights[(int64_t)next_blk * 16 + (tok & 15)];
            };
            fetch(first);
            for (int t = first; t < all; t += 2) {
                const int tok0 = begin + t * 128, tok = tok0 + row, blk = next_blk, n = seq + t;
                const float ks = next_ks, held = next_held;
                if (blk < 0 && tok < end && half == 0 && r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
                fetch(t + 2);
                float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
                if (t < act) {
                    const bool ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * odd, (n >> 1) & 1, &s_failed));
                    tc_fence_after();
                    const float2 ks2 = make_float2(ks, ks);
                    const bool edge = tok0 + 127 > least;
                    if (ok) {
#pragma unroll 1
                        for (int c = 0; c < HN / 32; ++c) {
                            uint32_t raw[32];
                            tc_ld32(from + 32 * c, raw);
                            const float4* f4 = reinterpret_cast<const float4*>(s_f + half * HN + 32 * c);
                            const float4* l4 = reinterpret_cast<const float4*>(s_nl + half * HN + 32 * c);
                            tc_wait_ld(raw);
                            if (c == HN / 32 - 1) {   // the buffer has been read
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(s_empty + 8 * odd);
                            }
                            float e[32];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float4 f = f4[i], l = l4[i];
                                const float2 a = __fmul2_rn(make_float2(f.x, f.y), ks2), d = __fmul2_rn(make_float2(f.z, f.w), ks2);
                                const float2 x = __ffma2_rn(make_float2(__uint_as_float(raw[4 * i]), __uint_as_float(raw[4 * i + 1])), a, make_float2(l.x, l.y));
                                const float2 y = __ffma2_rn(make_float2(__uint_as_float(raw[4 * i + 2]), __uint_as_float(raw[4 * i + 3])), d, make_float2(l.z, l.w));
                                e[4 * i] = ex2(x.x);
                                e[4 * i + 1] = ex2(x.y);
                                e[4 * i + 2] = ex2(y.x);
                                e[4 * i + 3] = ex2(y.y);
                            }
                            if (edge) {
                                asm volatile("" ::: "memory");   // few tiles: kept a branch
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (tok > s_lim[half * HN + 32 * c + i]) e[i] = 0.0f;
                            }
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                sum0 = __fadd2_rn(sum0, make_float2(e[4 * i], e[4 * i + 1]));
                                sum1 = __fadd2_rn(sum1, make_float2(e[4 * i + 2], e[4 * i + 3]));
                            }
                        }
                    }
                }
                float x = (sum0.x + sum0.y) + (sum1.x + sum1.y);
                if constexpr (C::TPT == 2) {   // a tile's 8 warps come here for each of their tiles, whatever became of their waits
                    if (half == 1) s_part[odd][(t >> 1) & 1][row] = x;
                    asm volatile("bar.sync %0, 256;" ::"r"(1 + odd) : "memory");
                    if (half == 0) x += s_part[odd][(t >> 1) & 1][row];
                }
                if (half == 0) {
                    if (chunk > 0) x += s_sum[tok - begin];
                    if (!last) s_sum[tok - begin] = x;
                    else if (blk >= 0) p.weights[(int64_t)blk * 16 + (tok & 15)] = tok < fresh && p.decay != 0.0f ? fmaf(p.decay, held, x) : x;
                }
            }
        } else if (warp == C::ISSUE) {
            // ── products ──
            if (rows > 0) {
                constexpr uint32_t id = mma_idesc(QN, 0);
                const uint32_t one = tc_elect();
                const uint64_t k_desc = tile_desc(k_at, 16), q = tile_desc(q_at, 16);
                bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, loads & 1, &s_failed));
                for (int t = 0; ok && t < act; ++t) {
                    const int n = seq + t, buf = n & 1;
                    ok = __all_sync(0xffffffffu, mbar_wait(k_full + 8 * buf, (n >> 1) & 1, &s_failed));
                    if (ok && n >= 2) ok = __all_sync(0xffffffffu, mbar_wait(s_empty + 8 * buf, ((n >> 1) & 1) ^ 1, &s_failed));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t k = k_desc + buf * (C::KTILE >> 4);
                    const uint32_t d = tmem + buf * QN;
#pragma unroll
                    for (int term = 0; term < 2; ++term)
#pragma unroll
                        for (int s = 0; s < D / 16; ++s)
                            tc_mma_ss(one, d, k + ((s >> 2) * (C::KSEG >> 4) + (s & 3) * 2),
                                      q + (term * (C::QTERM >> 4) + (s >> 2) * (C::QSEG >> 4) + (s & 3) * 2), id, term > 0 || s > 0);
                    tc_commit(one, s_full + 8 * buf);
                    tc_commit(one, k_empty + 8 * buf);
                }
            }
            __syncwarp();
        } else {
            // ── codes to tiles ──
            const int cw = warp - C::CONV, sub = lane >> 2, c4 = lane & 3;
            // codes are loaded a tile ahead, pages (lanes 0 .. 7: the tile's blocks) two
            uint4 w[C::UNITS][2];
            int blk = -1;
            auto locate = [&](int t) {
                const int tok = begin + t * 128 + lane * 16;
                blk = lane < 8 && t < act && tok < end ? block_at(r, b, h, tok >> 4) : -1;
            };
            auto load = [&]() {
#pragma unroll
                for (int u = 0; u < C::UNITS; ++u) {
                    const int unit = cw + C::CONV_WARPS * u, at = __shfl_sync(0xffffffffu, blk, (unit / C::SEGS) & 7);
                    w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
                    if (at >= 0 && unit < C::ALL_UNITS) {
                        const int8_t* from = r.k + (int64_t)at * (16 * D) + (unit % C::SEGS) * 64 + sub * D + 16 * c4;
                        w[u][0] = ldg_now(from);
                        w[u][1] = ldg_now(from + 8 * D);
                    }
                }
            };
            locate(0);
            load();
            locate(1);
            for (int t = 0; t < act; ++t) {
                const int n = seq + t, buf = n & 1;
                if (n >= 2 && !__all_sync(0xffffffffu, mbar_wait(k_empty + 8 * buf, ((n >> 1) & 1) ^ 1, &s_failed))) break;
#pragma unroll
                for (int u = 0; u < C::UNITS; ++u) {
                    const int unit = cw + C::CONV_WARPS * u, block = unit / C::SEGS, seg = unit % C::SEGS;
                    if (unit >= C::ALL_UNITS) break;
                    const uint32_t to = k_at + buf * C::KTILE + seg * C::KSEG + block * 2048 + sub * 128;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {   // rows sub and sub + 8 of the block
                        uint32_t o[8];
                        codes_to_f16(w[u][x], o);
                        sts128(to + x * 1024 + (((2 * c4) ^ sub) << 4), o[0], o[1], o[2], o[3]);
                        sts128(to + x * 1024 + (((2 * c4 + 1) ^ sub) << 4), o[4], o[5], o[6], o[7]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full + 8 * buf);
                load();
                locate(t + 2);
            }
        }
        seq += act;
        if (rows > 0) ++loads;
    }
    if (fail) break;
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

// A CTA's time is its tokens for each chunk of rows plus a start for each; one CTA an SM.  Its tokens at most fill the sums'
// place once where there are several chunks (beyond, it would read the rows again).
void weights_rows_plan(int64_t pairs, int D, int64_t rows, int64_t len, WeightsPlan* p) {
    const int qn = D == 128 ? WrCfg<128>::QN : WrCfg<256>::QN, sums = WrCfg<128>::TOKENS;
    const int64_t tile = 2 * (int64_t)qn * D * 2 + (int64_t)qn * sizeof(RowMeta), most = int64_t(1) << 30;
    p->rows = qn;
    p->chunks = (int)((rows + qn - 1) / qn);
    p->tiles = p->chunks;
    const int64_t pass = most / (tile * p->tiles);
    p->pairs_pass = (int)(pass < 1 ? 1 : (pass < pairs ? pass : pairs));
    p->bytes = (size_t)p->pairs_pass * p->tiles * tile;
    const int64_t slots = sm_count(), start = 512;
    int64_t best = INT64_MAX;
    for (int s = 1; s <= 256; ++s) {
        const int64_t per = ((len + s - 1) / s + 127) / 128 * 128;
        if (s > 1 && (int64_t)(s - 1) * per >= len) continue;
        const int64_t waves = (p->pairs_pass * s + slots - 1) / slots, turns = p->chunks > 1 ? (per + sums - 1) / sums : 1;
        const int64_t cost = waves * (per + start * turns);
        if (cost < best) { best = cost; p->splits = s; }
        if (waves > 8) break;
    }
}

template <int D>
static cudaError_t launch_weights_rows_d(const WeightsRun& r, const WeightsPlan& p, uint8_t* ws, cudaStream_t st) {
    using C = WrCfg<D>;
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = allow_smem(weights_rows_kernel<D>, C::SMEM, allowed);
    if (e != cudaSuccess) return e;
    RowMeta* meta = reinterpret_cast<RowMeta*>(ws + (size_t)p.pairs_pass * p.tiles * C::QTILE);
    const int64_t pairs = (int64_t)r.q.B * r.q.Hkv;
    for (int64_t pair0 = 0; pair0 < pairs; pair0 += p.pairs_pass) {
        const int now = (int)(pairs - pair0 < p.pairs_pass ? pairs - pair0 : p.pairs_pass);
        const int64_t warps = (int64_t)now * p.tiles * C::QN, grid = (int64_t)now * p.splits;
        if ((warps + 7) / 8 >= (int64_t(1) << 31) || grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
        weights_rows_prepare_kernel<D><<<(unsigned)((warps + 7) / 8), 256, 0, st>>>(r, pair0, now, p.tiles, ws, meta);
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
