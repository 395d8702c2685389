// tq_attn_q8.cu — attention over 8-bit pages for few query rows: decode steps and drafted tokens.
//
// For query row i of a sequence (i of q_len tokens) and the KV head of its group:
//   q' = H q (rotate_q),  s_j = sm_scale * sum_d q'_d c_jd * ks[j / 16],  p = softmax over the tokens it sees,
//   o = sum_j p_j c'_jd * vs[j / 16],  out = H o (v_rotated).
//
// Work.  A unit is up to 24 (D = 256: 16) query rows (tokens x heads of one group) of one (sequence, KV head); its
// tokens are split over CTAs, and within a CTA over 8 warps that never wait for one another: a warp takes every 8th
// block of 16 tokens (one scale block of K and V, 2 KB each at D = 128), which it copies into its own ring of
// shared memory (cp.async, 16 bytes a lane), converts once and multiplies with all rows of the unit.  Products are
// mma.sync m16n8k16 in f16 with fp32 accumulators, the cache as the A operand (16 tokens x 16 elements of K, 16
// elements x 16 tokens of V) and 8 rows as B: with the rows as A (16 of them), a decode step's 1 to 8 rows would
// leave half or more of every product empty, and accumulators, weights and query fragments would take twice the
// registers.  A tcgen05 tile (128 rows) would be emptier still, and its operands would have to go through shared
// memory once more after the conversion from 8 bits.
//
// What bounds it.  Single tokens: the cache's bytes, 16 sequences of 32768 tokens (1.08 GB) in 172 us, 6.25 TB/s, 95 % of
// the measured copy rate (ncu: DRAM 75 % of its nominal peak, integer pipe 55 %, issue 54 %).  From two or three
// groups of 8 rows on, the products' and exponentials' instructions and their latencies: 24 sequences of up to 9000
// tokens with 5 drafted tokens of 8 heads take 119 us, against 34 us for the bytes (issue 40 %, one CTA of 8 warps
// per SM by its 220 registers).  Short caches: the launches (9.7 us for one sequence of 1001 tokens).
//
// Numbers.  A row of q' is scaled by its largest element and rounded to f16; where the output has more than bf16's 8
// bits (LO) it is the sum of two f16 terms (float16 answers of 8 to 20 rows off by 2.4e-4 to 2.6e-4 of their norm
// instead of 4.1e-4, 2.1e-4 of it the output's rounding, in the same time).  Codes are integers of 8 bits and exact in
// f16.  K codes enter the product as subnormals (c + 128) 2^-24: one byte permute for two values;
// 128 times the row's sum of q' is taken off in fp32.  V codes are made from 1024 + (c + 128) minus 1152
// (the offset left in would cost up to 5 bits of the sum).  The V scale goes into the exponent:
// p_j = 2^(s_j + log2 vs - m + 6), so that one multiply-add per score applies both scales and every product is
// of f16 numbers near their row's largest, whatever the scales of other blocks; the sum of weights l takes
// p_j / vs in fp32.  m is the largest s + log2 vs seen up to a slack of 8: rows are rescaled only when a score
// exceeds m by more than that (p stays below 2^14, and is exact to f16's 11 bits down to 2^-20 of the largest).
#include <atomic>
#include <type_traits>
#include <utility>

#include "tq_attn_q8.cuh"
#include "tq_kernels.h"

namespace tq {

constexpr int Q8_WARPS = 8, Q8_THREADS = 32 * Q8_WARPS;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int D, int NT, bool LO> struct Q8Cfg {
    static constexpr int ROWS = 8 * NT, NK = D / 16;
    static constexpr int CTAS = D == 128 && NT == 1 ? 2 : 1;   // per SM
    static constexpr int STAGES = D == 256 || CTAS == 2 ? 3 : 5;
    static constexpr int BLOCK = 16 * D;                       // bytes of one tensor's block
    static constexpr int RING = STAGES * 2 * BLOCK;            // per warp
    static constexpr int QPART = NT * NK * 256, QBYTES = LO ? 2 * QPART : QPART;
    static constexpr int MERGE = Q8_WARPS * ROWS * D * 4;      // the warps' sums, over the rings
    static constexpr int RINGS = Q8_WARPS * RING > MERGE ? Q8_WARPS * RING : MERGE;
    static constexpr int SMEM = RINGS + QBYTES + (2 * Q8_WARPS * ROWS + 4 * ROWS) * 4;
};

// Four 8-bit codes of a word, biased by 128, as f16 subnormals (c + 128) 2^-24: elements 0, 1 and 2, 3.
__device__ __forceinline__ void bytes_sub(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;
    lo = __byte_perm(u, 0u, 0x4140);
    hi = __byte_perm(u, 0u, 0x4342);
}

// an 8 x 8 matrix of f16 pairs, transposed across the warp
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// One unit's share of tokens.  Partial results go to part / part_lse (splits > 1), else to out / lse.
template <int D, int NT, bool LO>
__global__ void __launch_bounds__(Q8_THREADS, Q8Cfg<D, NT, LO>::CTAS)
attn_q8_kernel(const Q8Run r, int row_tiles, int splits, float* __restrict__ part, float* __restrict__ part_lse) {
    using C = Q8Cfg<D, NT, LO>;
    constexpr int ROWS = C::ROWS, NK = C::NK, HALVES = D / 128, LPR = D / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* s_q = smem + C::RINGS;
    float* s_m = reinterpret_cast<float*>(s_q + C::QBYTES);   // [warp][row]
    float* s_l = s_m + Q8_WARPS * ROWS;
    // a row's factor of the scores (log2 domain, for sums of codes times 2^-24), and that of 128 * sum of its q'
    float2* s_f = reinterpret_cast<float2*>(s_l + Q8_WARPS * ROWS);
    int* s_lim = reinterpret_cast<int*>(s_f + ROWS);          // last token seen
    float* s_lse = reinterpret_cast<float*>(s_lim + ROWS);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int split = blockIdx.x % splits, rt = (blockIdx.x / splits) % row_tiles;
    const int pair = blockIdx.x / splits / row_tiles, h = pair % r.Hkv, b = pair / r.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const SeqLens sl = seq_lens(r, b);
    const int total_rows = (int)r.n * r.grp, row0 = rt * ROWS;

    // rows row0 .. of the unit: row i * grp + head of group.  The tokens that any of them sees: [0, kv_end)
    int last_i = (row0 + ROWS - 1) / r.grp;
    if (last_i >= sl.q_len) last_i = sl.q_len - 1;
    const int first_i = row0 / r.grp;
    const int kv_end = last_i < first_i ? 0 : last_seen(r, sl, last_i) + 1;
    const int per = ((kv_end + splits - 1) / splits + 127) & ~127;
    const int64_t begin64 = (int64_t)split * per;
    const int begin = begin64 < kv_end ? (int)begin64 : kv_end;
    const int end = kv_end - begin < per ? kv_end : begin + per;
    const int64_t unit = (int64_t)pair * row_tiles + rt;
    if (begin >= end && splits > 1) {
        if (threadIdx.x < ROWS) part_lse[(unit * splits + split) * ROWS + threadIdx.x] = -INFINITY;
        return;
    }

    // ── this warp's blocks; the first copies go out before q' is prepared ──
    const int nblk_all = (end - begin + 15) >> 4, blk0 = begin >> 4;
    const int mine = nblk_all > warp ? (nblk_all - warp + Q8_WARPS - 1) / Q8_WARPS : 0;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * C::RING;
    int nx_blk = -1, cu_blk = -1;                             // windows of 32 blocks, one per lane
    float nx_ks = 0.0f, nx_vs = 0.0f, cu_ks = 0.0f, cu_lv = 0.0f, cu_iv = 0.0f;
    auto window = [&](int i) {                                // blocks i .. i + 31 of this warp
        nx_blk = -1;
        nx_ks = nx_vs = 0.0f;
        if (i + lane < mine) {
            nx_blk = block_at(r, b, h, blk0 + warp + (i + lane) * Q8_WARPS);
            if (nx_blk >= 0) {
                nx_ks = r.ks[nx_blk];
                nx_vs = r.vs[nx_blk];
            } else if (r.status) {
                atomicMax(r.status, 1);
            }
        }
    };
    // A block's 16-byte chunk c of token x in a 128-byte half is copied to chunk c ^ (x & 7) of half * 2048 + x * 128.
    // A lane takes every 32nd chunk of the block; its places differ by constants and by the xor of constants.
    const uint32_t to0 = D == 128 ? (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4)
                                  : ((lane >> 3) & 1) * 2048 + (lane >> 4) * 128 + (((lane & 7) ^ (lane >> 4)) << 4);
    uint32_t fill = ring;                                     // the stage that the next copies go to
    auto issue = [&](int i) {
        if (i < mine) {
            if ((i & 31) == 0) window(i);
            const int blk = __shfl_sync(0xffffffffu, nx_blk, i & 31);
            if (blk >= 0) {
                const int8_t* kp = r.k + (int64_t)blk * C::BLOCK + lane * 16;
                const int8_t* vp = r.v + (int64_t)blk * C::BLOCK + lane * 16;
#pragma unroll
                for (int e = 0; e < C::BLOCK / 512; ++e) {
                    const uint32_t to = fill + e * (D == 128 ? 512 : 256) + (to0 ^ (D == 128 ? (e & 1) << 6 : ((2 * e) & 7) << 4));
                    cp16(to, kp + e * 512);
                    cp16(to + C::BLOCK, vp + e * 512);
                }
            }
        }
        cp_commit();
        fill += 2 * C::BLOCK;
        if (fill == ring + C::RING) fill = ring;
    };
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; ++i) issue(i);

    // ── q': Hadamard, row maximum, f16, in the order of the mma's B fragments ──
    // k-step j = 8 half + jj of lane t covers elements 128 half + 32 t + 4 jj .. + 3 (so that a lane's K bytes
    // are one run of 32), words b0, b1 = elements 0..1, 2..3 of row g; two k-steps in 16 bytes
    for (int base = warp * (32 / LPR); base < ROWS; base += Q8_WARPS * (32 / LPR)) {
        const int row = base + lane / LPR, e0 = (lane % LPR) * 16;
        const int gr = row0 + row, i = gr / r.grp;
        float v[16];
        const bool live = gr < total_rows && i < sl.q_len;
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
        const float inv = top >= 0x1p-100f ? __fdiv_rn(1.0f, top) : 0.0f;
        float sum = 0.0f;
        uint32_t w[8], wl[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = v[2 * j] * inv, y = v[2 * j + 1] * inv;
            const __half2 p = __floats2half2_rn(x, y);
            w[j] = *reinterpret_cast<const uint32_t*>(&p);
            sum += __low2float(p) + __high2float(p);
            if constexpr (LO) {   // what the rounding left, as a second term
                const __half2 q = __floats2half2_rn(x - __low2float(p), y - __high2float(p));
                wl[j] = *reinterpret_cast<const uint32_t*>(&q);
                sum += __low2float(q) + __high2float(q);
            }
        }
#pragma unroll
        for (int o = 1; o < LPR; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int half = e0 >> 7, tt = (e0 & 127) >> 5, j0 = half * 8 + ((e0 & 31) >> 2);
        uint4* to = reinterpret_cast<uint4*>(s_q) + ((row >> 3) * (NK / 2) + j0 / 2) * 32 + (row & 7) * 4 + tt;
        to[0] = make_uint4(w[0], w[1], w[2], w[3]);
        to[32] = make_uint4(w[4], w[5], w[6], w[7]);
        if constexpr (LO) {
            to[C::QPART / 16] = make_uint4(wl[0], wl[1], wl[2], wl[3]);
            to[C::QPART / 16 + 32] = make_uint4(wl[4], wl[5], wl[6], wl[7]);
        }
        if (lane % LPR == 0) {
            const float fr = top * r.sm_scale * LOG2E;
            s_f[row] = make_float2(fr * 0x1p24f, fr * 128.0f * sum);
            s_lim[row] = live ? last_seen(r, sl, i) : -1;
        }
    }
    __syncthreads();

    const uint32_t sq = (uint32_t)__cvta_generic_to_shared(s_q) + lane * 16;
    // this lane's rows: columns 2t and 2t + 1 of each n-tile
    float m[NT][2], l[NT][2];
    int lim_min = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = nt * 8 + 2 * t + e;
            lim_min = s_lim[row] < lim_min ? s_lim[row] : lim_min;
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.0f;
        }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);
    float o[NT][NK][4];   // m-tile i: elements 16 g + 2 i (words 0, 1) and 16 g + 2 i + 1 (words 2, 3) of each half
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.0f;

    // ── blocks of 16 tokens ──
    uint32_t kt = ring - 2 * C::BLOCK;
    for (int i = 0; i < mine; ++i) {
        cp_wait<C::STAGES - 2>();
        __syncwarp();
        if ((i & 31) == 0) {
            const float vse = nx_vs > 0.0f ? nx_vs : Q8_ZERO_SCALE;
            cu_blk = nx_blk;
            cu_ks = nx_ks;
            cu_lv = lg2(vse);
            cu_iv = __frcp_rn(vse);
        }
        issue(i + C::STAGES - 1);   // into the stage that was read in the last turn
        kt += 2 * C::BLOCK;
        if (kt == ring + C::RING) kt = ring;
        if (__shfl_sync(0xffffffffu, cu_blk, i & 31) < 0) continue;   // a page outside the pool holds nothing
        const float ks = __shfl_sync(0xffffffffu, cu_ks, i & 31), lv = __shfl_sync(0xffffffffu, cu_lv, i & 31);
        const float iv = __shfl_sync(0xffffffffu, cu_iv, i & 31);
        const uint32_t vt = kt + C::BLOCK;

        // scores: words 0, 1 of token g, words 2, 3 of token g + 8, for this lane's rows
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
            uint32_t kw[2][8];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t row = kt + half * 2048 + (x * 8 + g) * 128;
                const uint4 u = lds128(row + (((2 * t) ^ g) << 4)), w = lds128(row + (((2 * t + 1) ^ g) << 4));
                kw[x][0] = u.x; kw[x][1] = u.y; kw[x][2] = u.z; kw[x][3] = u.w;
                kw[x][4] = w.x; kw[x][5] = w.y; kw[x][6] = w.z; kw[x][7] = w.w;
            }
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                uint32_t a0[4], a1[4];
                bytes_sub(kw[0][j], a0[0], a0[2]);
                bytes_sub(kw[1][j], a0[1], a0[3]);
                bytes_sub(kw[0][j + 1], a1[0], a1[2]);
                bytes_sub(kw[1][j + 1], a1[1], a1[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint4 q = lds128(sq + (nt * (NK / 2) + half * 4 + j / 2) * 512);
                    mma16816(s[nt], a0, q.x, q.y);
                    mma16816(s[nt], a1, q.z, q.w);
                    if constexpr (LO) {
                        const uint4 ql = lds128(sq + C::QPART + (nt * (NK / 2) + half * 4 + j / 2) * 512);
                        mma16816(s[nt], a0, ql.x, ql.y);
                        mma16816(s[nt], a1, ql.z, ql.w);
                    }
                }
            }
        }

        // y = s * f ks + log2 vs
        const int tok0 = (blk0 + warp + i * Q8_WARPS) << 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float4 fr = *reinterpret_cast<const float4*>(s_f + nt * 8 + 2 * t);   // rows 2t and 2t + 1
            const float a0 = fr.x * ks, c0 = fmaf(-fr.y, ks, lv), a1 = fr.z * ks, c1 = fmaf(-fr.w, ks, lv);
            s[nt][0] = fmaf(s[nt][0], a0, c0);
            s[nt][1] = fmaf(s[nt][1], a1, c1);
            s[nt][2] = fmaf(s[nt][2], a0, c0);
            s[nt][3] = fmaf(s[nt][3], a1, c1);
        }
        if (tok0 + 15 > lim_min) {
            // the last blocks only: kept a branch
            asm volatile("" ::: "memory");
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int left = s_lim[nt * 8 + 2 * t + e] - tok0 - g;   // last token seen, from this lane's first
                    if (left < 0) s[nt][e] = -INFINITY;
                    if (left < 8) s[nt][2 + e] = -INFINITY;
                }
        }
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) over |= fmaxf(s[nt][e], s[nt][2 + e]) > m[nt][e] + Q8_SLACK;
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float now = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, x));
                    now = fmaxf(m[nt][e], now);
                    const float w = now == -INFINITY ? 1.0f : ex2(m[nt][e] - now);
                    m[nt][e] = now;
                    l[nt][e] *= w;
#pragma unroll
                    for (int j = 0; j < NK; ++j) {
                        o[nt][j][e] *= w;
                        o[nt][j][2 + e] *= w;
                    }
                }
        }
        uint32_t pf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float ref = m[nt][e] == -INFINITY ? 0.0f : m[nt][e] - Q8_SHIFT;
                p[e] = ex2(s[nt][e] - ref);
                p[2 + e] = ex2(s[nt][2 + e] - ref);
                l[nt][e] = fmaf(p[e] + p[2 + e], iv, l[nt][e]);
            }
            pf[nt][0] = transposed(pack_h2(p[0], p[1]));   // row g, tokens 2t, 2t + 1
            pf[nt][1] = transposed(pack_h2(p[2], p[3]));   // tokens 2t + 8, 2t + 9
        }

        // out += V^T P: the lane's elements 16 g .. 16 g + 15 of each half, tokens 2t, 2t + 1, 2t + 8, 2t + 9
        const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1152
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
            uint32_t vw[4][4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int row = 2 * t + (x & 1) + 8 * (x >> 1);
                const uint4 w = lds128(vt + half * 2048 + row * 128 + ((g ^ (row & 7)) << 4));
                vw[x][0] = w.x ^ 0x80808080u; vw[x][1] = w.y ^ 0x80808080u;
                vw[x][2] = w.z ^ 0x80808080u; vw[x][3] = w.w ^ 0x80808080u;
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {   // elements 4 w + 2 x and the next
                    const uint32_t sel = x ? 0x7362 : 0x5140;   // byte pairs (token 2t, 2t + 1) of two elements
                    const uint32_t lo = __byte_perm(vw[0][w], vw[1][w], sel), hi = __byte_perm(vw[2][w], vw[3][w], sel);
                    uint32_t a[4] = {__byte_perm(lo, 0x64646464u, 0x4140), __byte_perm(lo, 0x64646464u, 0x4342),
                                     __byte_perm(hi, 0x64646464u, 0x4140), __byte_perm(hi, 0x64646464u, 0x4342)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __half2 hv = __hsub2(*reinterpret_cast<__half2*>(&a[e]), off);
                        a[e] = *reinterpret_cast<const uint32_t*>(&hv);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][half * 8 + 2 * w + x], a, pf[nt][0], pf[nt][1]);
                }
            }
        }
    }
    cp_wait<0>();

    // ── the 8 warps' sums ──
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = l[nt][e];
#pragma unroll
            for (int y = 4; y < 32; y *= 2) x += __shfl_xor_sync(0xffffffffu, x, y);
            if (g == 0) {
                s_m[warp * ROWS + nt * 8 + 2 * t + e] = m[nt][e];
                s_l[warp * ROWS + nt * 8 + 2 * t + e] = x;
            }
        }
    __syncthreads();   // every warp is done with its ring
    // chunk c (4 floats) of a row at (c & ~7) | ((c ^ (row >> 1)) & 7): no bank conflicts
    float* sums = reinterpret_cast<float*>(smem);
    auto cell = [&](int w, int row, int c) {
        return sums + ((w * ROWS + row) * (D / 4) + ((c & ~7) | ((c ^ (row >> 1)) & 7))) * 4;
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int half = 0; half < HALVES; ++half)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int j = half * 8 + 2 * c;
                    *reinterpret_cast<float4*>(cell(warp, nt * 8 + 2 * t + e, half * 32 + 4 * g + c)) =
                        make_float4(o[nt][j][e], o[nt][j][2 + e], o[nt][j + 1][e], o[nt][j + 1][2 + e]);
                }
    __syncthreads();
    for (int id = threadIdx.x; id < ROWS * (D / 4); id += Q8_THREADS) {
        const int row = id / (D / 4), c = id % (D / 4);
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < Q8_WARPS; ++w) top = fmaxf(top, s_m[w * ROWS + row]);
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
        if (top != -INFINITY) {
#pragma unroll
            for (int w = 0; w < Q8_WARPS; ++w) {
                const float e = ex2(s_m[w * ROWS + row] - top);
                const float4 x = *reinterpret_cast<const float4*>(cell(w, row, c));
                sum = fmaf(s_l[w * ROWS + row], e, sum);
                a.x = fmaf(x.x, e, a.x); a.y = fmaf(x.y, e, a.y); a.z = fmaf(x.z, e, a.z); a.w = fmaf(x.w, e, a.w);
            }
            const float inv = __fdiv_rn(1.0f, sum);
            a.x *= inv; a.y *= inv; a.z *= inv; a.w *= inv;
        }
        const float lse = top == -INFINITY ? -INFINITY : (top - Q8_SHIFT + lg2(sum)) * LN2;
        if (splits > 1) {
            const int64_t at = (unit * splits + split) * ROWS + row;
            reinterpret_cast<float4*>(part + at * D)[c] = a;
            if (c == 0) part_lse[at] = lse;
        } else {
            // back to shared memory, in place of warp 0's sums (this thread has read them all)
            *reinterpret_cast<float4*>(cell(0, row, c)) = a;
            if (c == 0) s_lse[row] = lse;
        }
    }
    if (splits > 1) return;
    __syncthreads();
    for (int base = warp * (32 / LPR); base < ROWS; base += Q8_WARPS * (32 / LPR)) {
        const int row = base + lane / LPR, e0 = (lane % LPR) * 16, gr = row0 + row, i = gr / r.grp;
        float v[16];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4 x = *reinterpret_cast<const float4*>(cell(0, row, e0 / 4 + c));
            v[4 * c] = x.x; v[4 * c + 1] = x.y; v[4 * c + 2] = x.z; v[4 * c + 3] = x.w;
        }
        if (r.v_rotated) fwht16<D>(v, r.norm);
        if (gr < total_rows) {
            const int hq = h * r.grp + gr % r.grp;
            store_row16(r.out_dtype, r.out, b * r.os[0] + hq * r.os[1] + (int64_t)i * r.os[2] + e0, v);
            if (r.lse && e0 == 0) r.lse[((int64_t)b * r.Hq + hq) * r.n + i] = s_lse[row];
        }
    }
}

// Merge of the splits' normalized partial rows by their log-sum-exp, in split order, then the Hadamard
// transform and the output type, for `pairs` pairs from pair0 on.  D / 16 lanes take a row.
template <int D>
__global__ void __launch_bounds__(128) attn_q8_merge_kernel(const Q8Run r, int64_t pair0, int pairs, int rows, int row_tiles,
                                                            int splits, const float* __restrict__ part,
                                                            const float* __restrict__ part_lse) {
    constexpr int LPR = D / 16, RPC = 128 / LPR;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int total_rows = (int)r.n * r.grp;
    const int64_t all = (int64_t)pairs * total_rows;
    const int64_t id = (int64_t)blockIdx.x * RPC + threadIdx.x / LPR;
    const int e0 = (threadIdx.x % LPR) * 16;
    const int64_t slot = id < all ? id / total_rows : 0, pair = pair0 + slot;
    const int gr = id < all ? (int)(id - slot * total_rows) : 0;
    const int64_t unit = slot * row_tiles + gr / rows;
    const float* pl = part_lse + unit * splits * rows + gr % rows;
    float top = -INFINITY;
    for (int s = 0; s < splits; ++s) top = fmaxf(top, pl[(int64_t)s * rows]);
    float v[16], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0.0f;
    if (top != -INFINITY) {
        for (int s = 0; s < splits; ++s) {
            const float ls = pl[(int64_t)s * rows];
            if (ls == -INFINITY) continue;
            const float w = ex2((ls - top) * LOG2E);
            sum += w;
            const float4* x = reinterpret_cast<const float4*>(part + ((unit * splits + s) * rows + gr % rows) * D + e0);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float4 y = x[c];
                v[4 * c] = fmaf(w, y.x, v[4 * c]); v[4 * c + 1] = fmaf(w, y.y, v[4 * c + 1]);
                v[4 * c + 2] = fmaf(w, y.z, v[4 * c + 2]); v[4 * c + 3] = fmaf(w, y.w, v[4 * c + 3]);
            }
        }
        const float inv = __fdiv_rn(1.0f, sum);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] *= inv;
    }
    if (r.v_rotated) fwht16<D>(v, r.norm);
    if (id >= all) return;
    const int h = (int)(pair % r.Hkv), b = (int)(pair / r.Hkv), i = gr / r.grp, hq = h * r.grp + gr % r.grp;
    store_row16(r.out_dtype, r.out, b * r.os[0] + hq * r.os[1] + (int64_t)i * r.os[2] + e0, v);
    if (r.lse && e0 == 0) r.lse[((int64_t)b * r.Hq + hq) * r.n + i] = top == -INFINITY ? -INFINITY : top + lg2(sum) * LN2;
}

// ── plan and launch ────────────────────────────────────────────────────────

// Which kernel, by the query rows of a KV head (us at 8 sequences x 8 KV heads x 16000 tokens, D = 128 | 256):
//   rows         24          48          64         128          256         384         512
//   few       80 | 186   139 | 263   210 | 356   400 | 647   683 | 1243  947 | 1922  1345 | 2447
//   direct   121 | 233   130 | 239   124 | 238   129 | 241   226 |  439   349 | 668   446 |  874
//   tiles    303 | 470   305 | 470   303 | 471   306 | 475   290 |  577   433 | 831   399 |  868
// few: this file's kernel (a conversion for 24 or 16 rows); direct: tcgen05, a conversion for 128 rows; tiles:
// tcgen05 from tiles expanded once.  The bounds look at rows alone, so they lie between the crossings of different
// batches: at 48 rows of 128 the table has direct 7 % ahead, with 40 rows in 24 sequences of up to 9000 tokens few is
// (119 and 147 us).
constexpr int DIRECT_ROWS_128 = 49, DIRECT_ROWS_256 = 33, PROMPT_ROWS = 449;

// lo: q' as the sum of two f16 terms
Q8Plan q8_plan(int B, int Hkv, int grp, int D, int64_t n, int64_t max_len, bool lo) {
    Q8Plan p;
    p.lo = lo;
    const int64_t rows = n * grp, len = max_len > 0 ? max_len : 1;
    if (rows == 0 || B == 0) return p;
    p.prompt = rows >= (D == 128 ? DIRECT_ROWS_128 : DIRECT_ROWS_256);
    p.direct = rows < PROMPT_ROWS;
    // pairs that run at a time: where the work memory does not hold all pairs' tiles, the passes follow one another,
    // and rows and splits have to fill the SMs in each (72 pairs of 480 rows behind up to 131072 tokens run 15 at a
    // time: planned for all 72 at once they were 5 passes of 30 CTAs)
    p.pairs_pass = B * Hkv;
    if (p.prompt && !p.direct) q8_prompt_tiles((int64_t)B * Hkv, D, len, &p);
    if (p.prompt) {
        p.rows = q8_prompt_rows(p.pairs_pass, rows, D, p.direct, lo);
        p.row_tiles = (int)((rows + p.rows - 1) / p.rows);
    } else {
        // As few units as the registers allow, alike in size.  More rows share a conversion, but 40 of them leave
        // registers for 8 warps per SM only: 24 sequences of 5 x 8 rows, up to 9000 tokens: 131 us with 40, 118 to
        // 128 us with 24, 130 us with 16.
        const int most = D == 128 ? 24 : 16;
        p.row_tiles = (int)((rows + most - 1) / most);
        p.rows = (int)((rows + 8 * p.row_tiles - 1) / (8 * p.row_tiles)) * 8;
    }
    const int64_t units = (int64_t)p.pairs_pass * p.row_tiles;
    const int64_t slots = (int64_t)sm_count() * (D == 128 && p.rows == 8 ? 2 : 1);
    // Splits: a CTA's time is its tokens plus a start worth `start` tokens and, when split, the writing and merging of
    // its partial rows worth `join`; the grid runs in waves of `slots` CTAs.  Take the number with the least
    // waves * (tokens + start).  Two CTAs share an SM and hide each other's starts where units have 8 rows
    // (16 x 32768 tokens: 172 us with 1024, 179 us with 384); with one CTA per SM, lengths that differ want more and
    // shorter splits (24 sequences of up to 9000 tokens, 40 rows: 118 us with 384, 129 us with 1024).
    const int64_t start = p.prompt ? 768 : (slots > sm_count() ? 1024 : 384), join = p.prompt ? 512 : 0;
    int64_t best = INT64_MAX;
    for (int s = 1; s <= 256; ++s) {
        const int64_t per = ((len + s - 1) / s + 127) / 128 * 128;
        if (s > 1 && (int64_t)(s - 1) * per >= len) continue;   // the last split would be empty
        const int64_t waves = (units * s + slots - 1) / slots, cost = waves * (per + start + (s > 1 ? join : 0));
        if (cost < best) { best = cost; p.splits = s; }
        if (waves > 8) break;   // finer splits only add starts
    }
    return p;
}

// work memory of one pass: the splits' partial rows and their lse, then a prompt's tiles
static size_t part_rows(const Q8Plan& p) { return (size_t)p.pairs_pass * p.row_tiles * p.splits * p.rows; }
static size_t part_bytes(int D, const Q8Plan& p) {
    if (p.splits <= 1) return 0;
    return (part_rows(p) * (D + 1) * 4 + 255) & ~size_t(255);
}
size_t q8_workspace_bytes(int D, const Q8Plan& p) { return part_bytes(D, p) + p.tile_bytes; }

template <int D, int NT, bool LO>
static cudaError_t launch_one(const Q8Run& r, const Q8Plan& p, float* part, float* part_lse, cudaStream_t st) {
    using C = Q8Cfg<D, NT, LO>;
    cudaError_t e = cudaFuncSetAttribute(attn_q8_kernel<D, NT, LO>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    const int64_t grid = (int64_t)r.B * r.Hkv * p.row_tiles * p.splits;
    if (grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    attn_q8_kernel<D, NT, LO><<<(unsigned)grid, Q8_THREADS, C::SMEM, st>>>(r, p.row_tiles, p.splits, part, part_lse);
    return cudaGetLastError();
}

template <int D, int NT>
static cudaError_t launch_rows(const Q8Run& r, const Q8Plan& p, float* part, float* part_lse, cudaStream_t st) {
    return p.lo ? launch_one<D, NT, true>(r, p, part, part_lse, st) : launch_one<D, NT, false>(r, p, part, part_lse, st);
}

// raised by calls that bring no status word of their own; zero when the module is loaded
__device__ int32_t q8_status_word;

// its address on the current device (asked for once a device; the first call may be a captured one)
cudaError_t q8_default_status(int32_t** word) {
    static std::atomic<int32_t*> known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool keep = dev >= 0 && dev < 64;
    if (keep && (*word = known[dev].load(std::memory_order_relaxed)) != nullptr) return cudaSuccess;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if ((e = cudaThreadExchangeStreamCaptureMode(&mode)) != cudaSuccess) return e;
    void* at = nullptr;
    e = cudaGetSymbolAddress(&at, q8_status_word);
    const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess || back != cudaSuccess) return e != cudaSuccess ? e : back;
    *word = static_cast<int32_t*>(at);
    if (keep) known[dev].store(*word, std::memory_order_relaxed);
    return cudaSuccess;
}

cudaError_t launch_q8_merge(const Q8Run& r, const Q8Plan& p, int64_t pair0, int pairs, const float* part, const float* part_lse,
                            cudaStream_t st) {
    const int64_t rows = (int64_t)pairs * r.grp * r.n, rpc = 128 / (r.D / 16);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((rows + rpc - 1) / rpc));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (r.D == 256) return cudaLaunchKernelEx(&cfg, attn_q8_merge_kernel<256>, r, pair0, pairs, p.rows, p.row_tiles, p.splits, part, part_lse);
    return cudaLaunchKernelEx(&cfg, attn_q8_merge_kernel<128>, r, pair0, pairs, p.rows, p.row_tiles, p.splits, part, part_lse);
}

cudaError_t launch_attention_q8(const Q8Run& r, const Q8Plan& p, void* workspace, cudaStream_t st) {
    float* part = static_cast<float*>(workspace);
    float* part_lse = part + part_rows(p) * r.D;
    cudaError_t e;
    if (p.prompt) return launch_attention_q8_prompt(r, p, part, part_lse, static_cast<uint8_t*>(workspace) + part_bytes(r.D, p), st);
    if (r.D == 256) e = p.rows == 8 ? launch_rows<256, 1>(r, p, part, part_lse, st) : launch_rows<256, 2>(r, p, part, part_lse, st);
    else if (p.rows == 8) e = launch_rows<128, 1>(r, p, part, part_lse, st);
    else if (p.rows == 16) e = launch_rows<128, 2>(r, p, part, part_lse, st);
    else e = launch_rows<128, 3>(r, p, part, part_lse, st);
    if (e != cudaSuccess || p.splits <= 1) return e;
    return launch_q8_merge(r, p, 0, p.pairs_pass, part, part_lse, st);
}

}  // namespace tq
