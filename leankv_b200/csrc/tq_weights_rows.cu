// tq_weights_rows.cu — sums of attention weights over 8-bit keys for many query rows (prompts, windows of them), on tcgen05.
//
// The mathematics is tq_weights.cu's.  With many rows per KV head the products and the exponentials bound it, not the keys.
// Scores are computed as K Q^T, tokens on the lanes of TMEM and query rows on its columns: a thread then adds up the weights of
// its token over the columns that it reads, with nothing to exchange, and tokens' sums leave the kernel as one float.
//
// weights_rows_prepare_kernel: q' (Hadamard, row maximum) as two f16 terms, into images of the shared-memory tiles, once per call
// (a row is read by every CTA of its KV head); with each row's factor, log-sum-exp and last token.
//
// weights_rows_kernel: a CTA takes a run of tokens of one (sequence, KV head) and CH rows at a time, whose tiles stay in shared
// memory while the run's keys come by, 128 tokens at a time.  Warps:
//   4      convert codes to f16 tiles (two buffers)
//   1      issues the products: S = K (Q1 + Q2)^T, 128 tokens x QN rows, f16, fp32 sums in TMEM
//   2 x 4  take turns at the tokens' tiles: scores from TMEM, weights, sums
// More rows than CH are taken in turn, the run's sums kept in shared memory between.  Row tiles whose rows see none of a tile's
// tokens (prompts' later halves) are left out.
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
    static constexpr int QN = D == 128 ? 128 : 64, NQ = D == 128 ? 2 : 1, CH = QN * NQ;   // rows of a tile, tiles, rows at a time
    static constexpr int SEGS = D / 64;
    static constexpr int QTERM = QN * D * 2, QTILE = 2 * QTERM;                           // bytes
    static constexpr int KTILE = 128 * D * 2, KSEG = 128 * 128, QSEG = QN * 128;
    static constexpr int EPI = 8, ISSUE = EPI, CONV = EPI + 1, CONV_WARPS = 4, WARPS = CONV + CONV_WARPS, THREADS = 32 * WARPS;
    static constexpr int UNITS = 8 * SEGS / CONV_WARPS;                                   // of a converting warp: 16 tokens x 64 elements
    static constexpr int TOKENS = 4096;                                                   // of a CTA at most
    static constexpr int SMEM = 1024 + NQ * QTILE + 2 * KTILE + TOKENS * 4;
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
    constexpr int QN = C::QN, NQ = C::NQ;
    const Q8Run& r = p.q;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[16];
    __shared__ __align__(16) float s_f[C::CH], s_nl[C::CH];
    __shared__ int s_lim[C::CH], s_most[NQ], s_least[NQ];   // last tokens of the rows; the largest and the least of a tile's
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    uint8_t* tiles_at = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t q_at = smem_u32(tiles_at), k_at = q_at + NQ * C::QTILE, bar0 = smem_u32(bars);
    float* s_sum = reinterpret_cast<float*>(tiles_at + NQ * C::QTILE + 2 * C::KTILE);
    const uint32_t k_full = bar0, k_empty = bar0 + 16, s_full = bar0 + 32, s_empty = bar0 + 64, q_full = bar0 + 96, done = bar0 + 104;

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
    const int rows = (int)(sl.q_len > p.window ? p.window : sl.q_len) * r.grp, chunks = rows ? (rows + C::CH - 1) / C::CH : 1;

    if (threadIdx.x == 0) {
        s_failed = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, C::CONV_WARPS);
            mbar_init(k_empty + 8 * i, 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(s_empty + 8 * i, 4);
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

    // alike in all warps: tiles of keys so far; parity of the uses of the score buffers (group of the tile, row tile), and which
    // have been used; chunks of rows
    int seq = 0, loads = 0;
    uint32_t parity = 0, begun = 0;
    bool fail = false;
    const int step = chunks > 1 ? C::TOKENS : per;   // sums wait for the next chunk only
    for (int begin = begin_all; begin < end_all; begin += step) {
    const int end = end_all - begin < step ? end_all : begin + step, all = (end - begin + 127) >> 7;
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const bool last = chunk + 1 == chunks;
        const int nq = rows - chunk * C::CH >= C::CH ? NQ : (rows - chunk * C::CH + QN - 1) / QN;   // 0 without rows
        const int64_t tile0 = (int64_t)slot * tiles + chunk * NQ;
        // the rows before are no longer used (their products have been waited for); all leave together after a failed wait
        fail = __syncthreads_or(s_failed) != 0;
        if (fail) break;
        if (threadIdx.x == 0 && nq > 0) {
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(q_full), "r"(nq * C::QTILE) : "memory");
            for (int i = 0; i < 2 * nq; ++i)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(q_at + i * C::QTERM), "l"(images + tile0 * C::QTILE + i * C::QTERM), "r"(C::QTERM), "r"(q_full) : "memory");
        }
        for (int i = threadIdx.x; i < nq * QN; i += C::THREADS) {
            const RowMeta m = meta[tile0 * QN + i];
            s_f[i] = m.f;
            s_nl[i] = m.nl;
            s_lim[i] = m.lim;
        }
        __syncthreads();
        if (warp < nq) {
            int most = -1, least = 0x7fffffff;
            for (int i = lane; i < QN; i += 32) {
                const int x = s_lim[warp * QN + i];
                most = max(most, x);
                least = min(least, x < 0 ? 0x7fffffff : x);
            }
            most = __reduce_max_sync(0xffffffffu, most);
            least = __reduce_min_sync(0xffffffffu, least);
            if (lane == 0) {
                s_most[warp] = most;
                s_least[warp] = least;
            }
        }
        __syncthreads();
        // tiles of keys that some row of the row tile sees
        int seen[NQ], act = 0;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const int most = j < nq ? s_most[j] : -1;
            seen[j] = most < begin ? 0 : min(all, ((most - begin) >> 7) + 1);
            act = max(act, seen[j]);
        }

        if (warp < C::EPI) {
            // ── weights and sums: thread = token ──
            const int group = warp >> 2;
            const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            bool ok = true;
            for (int t = group; t < all; t += 2) {
                const int tok0 = begin + t * 128, tok = tok0 + (warp & 3) * 32 + lane;
                const int blk = tok < end ? block_at(r, b, h, tok >> 4) : -1;
                const float ks = blk >= 0 ? r.ks[blk] : 0.0f;
                float* at = p.weights + ((int64_t)blk * 16 + (tok & 15));
                float held = 0.0f;
                if (blk >= 0 && last && tok < fresh && p.decay != 0.0f) held = *at;
                if (blk < 0 && tok < end && r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
                float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
                const float2 ks2 = make_float2(ks, ks);
#pragma unroll
                for (int j = 0; j < NQ; ++j) {
                    if (t >= seen[j]) continue;
                    const int buf = group * NQ + j;
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(s_full + 8 * buf, (parity >> buf) & 1, &s_failed));
                    parity ^= 1u << buf;
                    if (!ok) break;
                    tc_fence_after();
                    const bool edge = tok0 + 127 > s_least[j];
#pragma unroll 1
                    for (int c = 0; c < QN / 32; ++c) {
                        uint32_t raw[32];
                        tc_ld32(lanes + buf * QN + 32 * c, raw);
                        const float4* f4 = reinterpret_cast<const float4*>(s_f + j * QN + 32 * c);
                        const float4* l4 = reinterpret_cast<const float4*>(s_nl + j * QN + 32 * c);
                        tc_wait_ld(raw);
                        if (c == QN / 32 - 1) {   // the buffer has been read
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(s_empty + 8 * buf);
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
                                if (tok > s_lim[j * QN + 32 * c + i]) e[i] = 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            sum0 = __fadd2_rn(sum0, make_float2(e[4 * i], e[4 * i + 1]));
                            sum1 = __fadd2_rn(sum1, make_float2(e[4 * i + 2], e[4 * i + 3]));
                        }
                    }
                }
                if (!ok) break;
                float x = (sum0.x + sum0.y) + (sum1.x + sum1.y);
                if (chunk > 0) x += s_sum[tok - begin];
                if (!last) s_sum[tok - begin] = x;
                else if (blk >= 0) *at = tok < fresh && p.decay != 0.0f ? fmaf(p.decay, held, x) : x;
            }
        } else if (warp == C::ISSUE) {
            // ── products ──
            if (nq > 0) {
                constexpr uint32_t id = mma_idesc(QN, 0);
                const uint32_t one = tc_elect();
                const uint64_t k_desc = tile_desc(k_at, 16), q_desc = tile_desc(q_at, 16);
                bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, loads & 1, &s_failed));
                for (int t = 0; ok && t < act; ++t) {
                    const int kb = (seq + t) & 1, group = t & 1;
                    ok = __all_sync(0xffffffffu, mbar_wait(k_full + 8 * kb, ((seq + t) >> 1) & 1, &s_failed));
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < NQ; ++j) {
                        if (!ok || t >= seen[j]) continue;
                        const int buf = group * NQ + j;
                        if ((begun >> buf) & 1) ok = __all_sync(0xffffffffu, mbar_wait(s_empty + 8 * buf, ((parity >> buf) & 1) ^ 1, &s_failed));
                        if (!ok) continue;
                        tc_fence_after();
                        parity ^= 1u << buf;
                        begun |= 1u << buf;
                        const uint64_t k = k_desc + kb * (C::KTILE >> 4), q = q_desc + j * (C::QTILE >> 4);
                        const uint32_t d = tmem + buf * QN;
#pragma unroll
                        for (int term = 0; term < 2; ++term)
#pragma unroll
                            for (int s = 0; s < D / 16; ++s)
                                tc_mma_ss(one, d, k + ((s >> 2) * (C::KSEG >> 4) + (s & 3) * 2),
                                          q + (term * (C::QTERM >> 4) + (s >> 2) * (C::QSEG >> 4) + (s & 3) * 2), id, term > 0 || s > 0);
                        tc_commit(one, s_full + 8 * buf);
                    }
                    if (ok) tc_commit(one, k_empty + 8 * kb);
                }
            }
            __syncwarp();
        } else {
            // ── codes to tiles ──
            const int cw = warp - C::CONV, sub = lane >> 2, c4 = lane & 3;
            uint4 w[C::UNITS][2];
            auto load = [&](int t) {
#pragma unroll
                for (int u = 0; u < C::UNITS; ++u) {
                    const int unit = cw + C::CONV_WARPS * u, block = unit / C::SEGS, seg = unit % C::SEGS, tok = begin + t * 128 + block * 16;
                    const int blk = tok < end ? block_at(r, b, h, tok >> 4) : -1;
                    w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
                    if (blk >= 0) {
                        const int8_t* from = r.k + (int64_t)blk * (16 * D) + seg * 64 + sub * D + 16 * c4;
                        w[u][0] = ldg_now(from);
                        w[u][1] = ldg_now(from + 8 * D);
                    }
                }
            };
            if (act > 0) load(0);
            for (int t = 0; t < act; ++t) {
                const int kb = (seq + t) & 1;
                if (seq + t >= 2 && !__all_sync(0xffffffffu, mbar_wait(k_empty + 8 * kb, (((seq + t) >> 1) & 1) ^ 1, &s_failed))) break;
#pragma unroll
                for (int u = 0; u < C::UNITS; ++u) {
                    const int unit = cw + C::CONV_WARPS * u, block = unit / C::SEGS, seg = unit % C::SEGS;
                    const uint32_t to = k_at + kb * C::KTILE + seg * C::KSEG + block * 2048 + sub * 128;
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
                if (lane == 0) mbar_arrive(k_full + 8 * kb);
                if (t + 1 < act) load(t + 1);
            }
        }
        seq += act;
        if (nq > 0) ++loads;
        // uses of the buffers that this warp has not counted itself
        if (warp != C::ISSUE) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int j = 0; j < NQ; ++j)
                    if (warp >= C::EPI || (warp >> 2) != g) parity ^= (uint32_t)(((seen[j] + 1 - g) >> 1) & 1) << (g * NQ + j);
        }
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
    const int qn = D == 128 ? WrCfg<128>::QN : WrCfg<256>::QN, ch = D == 128 ? WrCfg<128>::CH : WrCfg<256>::CH;
    const int64_t tile = 2 * (int64_t)qn * D * 2 + (int64_t)qn * sizeof(RowMeta), most = int64_t(1) << 30;
    p->rows = ch;
    p->chunks = (int)((rows + ch - 1) / ch);
    p->tiles = p->chunks * (ch / qn);
    const int64_t pass = most / (tile * p->tiles);
    p->pairs_pass = (int)(pass < 1 ? 1 : (pass < pairs ? pass : pairs));
    p->bytes = (size_t)p->pairs_pass * p->tiles * tile;
    const int64_t slots = sm_count(), start = 512;
    int64_t best = INT64_MAX;
    for (int s = 1; s <= 256; ++s) {
        const int64_t per = ((len + s - 1) / s + 127) / 128 * 128;
        if (s > 1 && (int64_t)(s - 1) * per >= len) continue;
        const int64_t waves = (p->pairs_pass * s + slots - 1) / slots, turns = p->chunks > 1 ? (per + 4095) / 4096 : 1;
        const int64_t cost = waves * (per + start * turns);
        if (cost < best) { best = cost; p->splits = s; }
        if (waves > 8) break;
    }
}

template <int D>
static cudaError_t launch_weights_rows_d(const WeightsRun& r, const WeightsPlan& p, uint8_t* ws, cudaStream_t st) {
    using C = WrCfg<D>;
    cudaError_t e = cudaFuncSetAttribute(weights_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
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
