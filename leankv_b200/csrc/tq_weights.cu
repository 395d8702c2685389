// tq_weights.cu — sums of the attention weights that cached tokens get from a step's queries, over 8-bit or TurboQuant keys.
//
// For token t of (sequence b, KV head h), over the group's query heads and the last `window` rows i of the sequence:
//   w[t] <- (t < fresh[b] ? decay * w[t] : 0) + sum over rows that see t of exp(s_it - lse_i),  s_it = sm_scale q'_i . k_t
// with the log-sum-exp that the attention of those rows has left.  V is not read, and no weight leaves the SM.
//
// Work.  A CTA takes a run of tokens of one (sequence, KV head); its 8 warps take every 8th block of 16 tokens, copied into
// a ring of the warp's own in shared memory (cp.async), their earlier weights with them.  Products are mma.sync with the keys as
// the A operand (16 tokens) and 8 query rows as B: a thread's sums over the rows are then sums over its columns, which four
// lanes add up at the end.  More than 32 rows of TurboQuant keys are taken 32 at a time, the tokens' sums kept in shared memory
// between; of 8-bit keys they go to tq_weights_rows.cu.  us with this file's kernel and with that one, 2 x 16000 tokens of 8 KV heads:
//   rows       32        36         64         128         256
//   D = 128    28     39 | 29    55 | 29    107 | 36    210 | 55
//   D = 256    50     68 | 35    95 | 36    186 | 45    367 | 76
// The bound of 32 rows is that of D = 128; heads of 256 with 32 rows would be faster there (about 35 us).
//
// What bounds it.  8 bits: the keys' bytes, 16 sequences of 32768 tokens of 8 KV heads (0.57 GB with the earlier weights) in 102 us,
// 5.6 TB/s (86 % of the measured copy rate; a fourth of them in 36 us: issue 60 %, integer pipe 34 %, DRAM 48 %).  With f16 products
// of converted codes the same took 129 us.  TurboQuant: instructions and their latency, 32 sequences of up to 9000 tokens
// of TQ3 keys in 54 us, floor 11 (8 of 9000 in 34 us: issue 59 %, integer pipe 47 %, DRAM 12 %); 60 us with pairs of levels as
// f16 terms from a table in shared memory (its wavefronts 61 %), 136 us with levels made by arithmetic.  32 other ragged sequences to
// 9000 tokens of 8 KV heads, one token of 64 heads, us for 8 bits, TQ4, TQ3, TQ2: heads of 128 42, 67, 59, 56; heads of 256 60, 134, 98, 90.
// More rows of 8-bit keys (16, 24, 32 rows over 16 x 9000 tokens of 8 KV heads): 59, 77, 92 us, of heads of 256 116, 148, 182: the
// products and powers of a tile of 8 rows.  One sequence of 1001 tokens: the launch, 4.7 us.
//
// Numbers.  Sums are fp32 results that later sums are added to, so scores are kept to fp32's size of error.
// 8 bits: codes enter s8 products (m16n8k32, exact in s32) as they lie in memory; a row of q' is scaled by its largest element
// and is the sum of three terms of 8 bits, q1 + q2 / 254 + q3 / 254^2 (2^-24 of the largest element).  In f16 the codes have to be
// converted and q' is two terms: as many operations on twice the instructions.  The sums start from the bits of 1.5 * 2^23, so that
// they are floats as they are (their size is below 2^22).
// TQ2, TQ3: levels are sums of three such terms, too, whose bytes a byte permute looks up four at a time; of the nine products of
// terms those below 2^-23 of the largest elements are left out, six remain.  TQ4 has more levels than a permute takes: its levels
// are the sum of two f16 terms, looked up by the pair in shared memory, and so is q'; m16n8k16, fp32 sums.
#include <type_traits>

#include "leankv_tq.h"
#include "tq_attn_q8.cuh"
#include "tq_evict.h"
#include "tq_kernels.h"
#include "tq_warp_rows.cuh"

namespace tq {

constexpr int WT_WARPS = 8, WT_THREADS = 32 * WT_WARPS, WT_ROWS = 32;   // most rows at a time
constexpr int WT_START = 1024;     // what a CTA's start is worth, in tokens (512 is slower for 8-bit keys, 2048 for TQ3 ones, 256 for both)
constexpr int WT_TOKENS = 2048;   // tokens of a CTA whose sums wait in shared memory

__device__ __forceinline__ void wt_cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 wt_lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 wt_lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ float wt_lds32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t wt_lds16(uint32_t a) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ int wt_lds16s(uint32_t a) {
    int16_t v;
    asm volatile("ld.shared.s16 %0, [%1];" : "=h"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void wt_imma(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the sums begin with this product, at `zero`
__device__ __forceinline__ void wt_imma_first(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int zero) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(zero));
}
__device__ __forceinline__ void wt_mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void wt_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The eight (TQ3) or four (TQ2) levels in units of 1/127 of the largest one, as the sum of three terms of 8 bits, l1 + l2 / 254 +
// l3 / 254^2: term k of levels 4 w .. 4 w + 3 in the bytes of a word.
template <int QT> constexpr uint32_t wt_levels(int k, int w) {
    uint32_t bytes = 0;
    for (int i = 0; i < 4; ++i) {
        double x = (double)tq_level<QT>((4 * w + i) & ((1 << QT) - 1)) / (double)tq_level<QT>((1 << QT) - 1) * 127.0;
        int term = 0;
        for (int j = 0; j <= k; ++j) {
            term = (int)(x < 0.0 ? x - 0.5 : x + 0.5);
            x = (x - term) * 254.0;
        }
        bytes |= (uint32_t)(term & 0xFF) << (8 * i);
    }
    return bytes;
}
__device__ __forceinline__ uint32_t wt_either(uint32_t mask, uint32_t a, uint32_t b) { return (a & mask) | (b & ~mask); }
// byte i of the result: byte (nibble i of s, 0 .. 7) of lo and hi
__device__ __forceinline__ uint32_t wt_prmt(uint32_t lo, uint32_t hi, uint32_t s) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(lo), "r"(hi), "r"(s));
    return d;
}

// TILES: tiles of 8 rows at a time, 1 or 4
template <int D, int QT, int TILES> struct WtCfg {
    static constexpr int NK = D / 16, ROWS = 8 * TILES;
    static constexpr int ROWB = QT == 8 ? D : D / 32 * BlockBytes<QT == 8 ? 4 : QT>::value;
    static constexpr int TILE = 16 * ROWB;                       // bytes of a block of 16 tokens
    static constexpr int STAGE = TILE + 64;                      // with their earlier weights
    static constexpr int STAGES = QT == 8 && D == 256 ? 3 : 4;
    static constexpr int RING = STAGES * STAGE;                  // per warp
    // q': 8 bits three terms, [tile][pair of k-steps][3][lane] of 16 bytes; TQ2 and TQ3 three terms, [tile][block of 32 elements], the first
    // two [lane] of 16 bytes and the third [lane] of 8; TQ4 two parts of [tile][pair of k-steps][lane]
    static constexpr int QPART = TILES * NK * 256, QBLOCK = 768, QBYTES = QT == 4 ? 2 * QPART : TILES * (D / 32) * QBLOCK;
    // TQ4: pairs of levels as f16 terms, an entry of 256 bytes, 8 for every lane, so that lookups do not meet in a bank and a lookup's
    // address is the pair's number in one byte and the lane's in the next
    static constexpr int PAIRS = QT == 4 ? 256 : 0, TABLE = PAIRS * 256;
    // what a sum of products counts: TQ2 and TQ3 levels are in units of 1/127 of the largest one, too
    static constexpr float UNIT = QT == 4 ? 1.0f : QT == 8 ? 1.0f / 127.0f : tq_level<QT == 8 ? 4 : QT>((1 << (QT & 3)) - 1) / (127.0f * 127.0f);
    static constexpr int SUMS = TILES > 1 ? WT_TOKENS * 4 : 0;   // tokens' sums between chunks of rows
    static constexpr int SMEM = TABLE + WT_WARPS * RING + QBYTES + SUMS;
    static constexpr int CTAS = SMEM <= 74 * 1024 ? 3 : SMEM <= 112 * 1024 ? 2 : 1;
};

// half_decode() in three operations: the bits moved to a float's place are the value times 2^-112, whatever the exponent
__device__ __forceinline__ float scale_decode(int h) {   // sign-extended, so that the sign is in its place, and in those of the exponent's top
    return __uint_as_float(((uint32_t)h << 13) & 0x8FFFFFFFu) * 0x1p112f;
}

template <int D, int QT, int TILES>
__global__ void __launch_bounds__(WT_THREADS, WtCfg<D, QT, TILES>::CTAS) weights_kernel(const WeightsRun p, int splits, int row_chunks) {
    using C = WtCfg<D, QT, TILES>;
    constexpr int NK = C::NK, ROWS = C::ROWS;
    const Q8Run& r = p.q;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* s_q = smem + C::TABLE + WT_WARPS * C::RING;   // the table comes first
    float* s_sum = reinterpret_cast<float*>(s_q + C::QBYTES);
    __shared__ __align__(16) float2 s_f[ROWS];      // a row's factor of the scores and its log-sum-exp, in the log2 domain
    __shared__ int s_lim[ROWS];                     // last token that it sees

    const int split = blockIdx.x % splits, pair = blockIdx.x / splits, h = pair % r.Hkv, b = pair / r.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const SeqLens sl = seq_lens(r, b);
    const int per = ((sl.len + splits - 1) / splits + 127) & ~127;
    const int64_t begin64 = (int64_t)split * per;
    if (begin64 >= sl.len) return;
    const int begin_all = (int)begin64, end_all = sl.len - begin_all < per ? sl.len : begin_all + per;
    const int fresh = p.fresh ? p.fresh[b] : 0x7fffffff;
    const int i0 = sl.q_len > p.window ? sl.q_len - (int)p.window : 0;
    const int rows_all = (sl.q_len - i0) * r.grp;   // rows i0 .. of the sequence, row = token x head of group

    if constexpr (QT == 4) {
        __shared__ float s_level[1 << (QT & 7)];
        if (threadIdx.x < (1 << QT)) {
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < (1 << QT); ++i)
                if (i == threadIdx.x) x = tq_level<QT>(i);
            s_level[threadIdx.x] = x;
        }
        __syncthreads();
        for (int i = warp; i < C::PAIRS; i += WT_WARPS) {   // two levels as the sum of two pairs of f16 terms
            const float x = s_level[i & ((1 << QT) - 1)], y = s_level[i >> QT];
            const __half2 hi = __floats2half2_rn(x, y);
            reinterpret_cast<uint2*>(smem)[i * 32 + lane] =
                make_uint2(*reinterpret_cast<const uint32_t*>(&hi), pack_h2(x - __low2float(hi), y - __high2float(hi)));
        }
    }

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + C::TABLE + warp * C::RING;
    const uint32_t sq = (uint32_t)__cvta_generic_to_shared(s_q) + lane * 16;
    const uint32_t lane8 = lane * 8;
    uint32_t levels[3][2];   // TQ2, TQ3
    if constexpr (QT == 2 || QT == 3) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            constexpr uint32_t w[3][2] = {{wt_levels<QT>(0, 0), wt_levels<QT>(0, 1)}, {wt_levels<QT>(1, 0), wt_levels<QT>(1, 1)},
                                          {wt_levels<QT>(2, 0), wt_levels<QT>(2, 1)}};
            levels[k][0] = w[k][0];
            levels[k][1] = w[k][1];
        }
    }

    // with several chunks of rows, as many tokens at a time as have sums in shared memory
    const int step = row_chunks > 1 ? WT_TOKENS : per;
    for (int begin = begin_all; begin < end_all; begin += step) {
    const int end = end_all - begin < step ? end_all : begin + step;
    const int nblk_all = (end - begin + 15) >> 4, blk0 = begin >> 4;
    const int mine = nblk_all > warp ? (nblk_all - warp + WT_WARPS - 1) / WT_WARPS : 0;
    for (int chunk = 0; chunk < row_chunks; ++chunk) {
        const int row0 = chunk * ROWS, rows = rows_all - row0 < ROWS ? rows_all - row0 : ROWS;
        const bool last = chunk + 1 == row_chunks || rows_all - row0 <= ROWS;
        const int tiles = TILES == 1 ? 1 : rows > 0 ? (rows + 7) >> 3 : 0;
        const bool reads = last && p.decay != 0.0f;   // the earlier weights, copied with the keys

        int nx_blk = -1, cu_blk = -1;                // windows of 32 blocks, one per lane
        float nx_ks = 0.0f, cu_ks = 0.0f;
        auto window = [&](int i) {
            nx_blk = -1;
            nx_ks = 0.0f;
            if (i + lane < mine) {
                nx_blk = block_at(r, b, h, blk0 + warp + (i + lane) * WT_WARPS);
                if (nx_blk < 0) {
                    if (r.status) atomicMax(r.status, (int)TQ_ERROR_INVALID_VALUE);
                } else if (QT == 8) {
                    nx_ks = r.ks[nx_blk];
                }
            }
        };
        // 8 bits: 16-byte chunk c of token x in a 128-byte half goes to chunk c ^ (x & 7) of half * 2048 + x * 128; a lane takes
        // every 32nd chunk of the block, and its places differ by constants and by the xor of constants
        const uint32_t to0 = QT != 8 ? lane * 16 : D == 128 ? (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4)
                                       : ((lane >> 3) & 1) * 2048 + (lane >> 4) * 128 + (((lane & 7) ^ (lane >> 4)) << 4);
        uint32_t fill = ring;
        auto issue = [&](int i) {
            if (i < mine) {
                if ((i & 31) == 0) window(i);
                const int blk = __shfl_sync(0xffffffffu, nx_blk, i & 31);
                if (blk >= 0) {
                    const int8_t* kp = r.k + (int64_t)blk * C::TILE + lane * 16;
#pragma unroll
                    for (int e = 0; e < (C::TILE + 511) / 512; ++e) {
                        uint32_t to = to0 + e * 512;
                        if constexpr (QT == 8) to = e * (D == 128 ? 512 : 256) + (to0 ^ (D == 128 ? (e & 1) << 6 : ((2 * e) & 7) << 4));
                        if (C::TILE % 512 == 0 || lane + 32 * e < C::TILE / 16) wt_cp16(fill + to, kp + e * 512);
                    }
                    if (reads && lane < 4) wt_cp16(fill + C::TILE + lane * 16, p.weights + (int64_t)blk * 16 + lane * 4);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            fill += C::STAGE;
            if (fill == ring + C::RING) fill = ring;
        };
        if (chunk > 0 || begin > begin_all) __syncthreads();   // the rows before have been used
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; ++i) issue(i);

        // ── q': Hadamard, row maximum, terms in the order of the products' B fragments; a warp takes a row ──
        for (int row = warp; row < tiles * 8; row += WT_WARPS) {
            constexpr int E = D / 32;
            const int e0 = lane * E, gr = row0 + row, i = i0 + gr / r.grp, hq = h * r.grp + gr % r.grp;
            float v[E];
            // a row that saw nothing adds nothing, whatever q holds there
            const float lse = row < rows ? p.lse[((int64_t)b * r.Hq + hq) * r.n + i] : -INFINITY;
            const bool sees = lse != -INFINITY;
            if (sees) {
                load_some<E>(r.q_dtype, r.q, b * r.qs[0] + hq * r.qs[1] + (int64_t)i * r.qs[2] + e0, v);
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j) v[j] = 0.0f;
            }
            if (r.rotate_q) fwht_warp<E>(v, r.norm);
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < E; ++j) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
            for (int o = 1; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float inv = top >= 0x1p-100f ? __fdiv_rn(QT == 4 ? 1.0f : 127.0f, top) : 0.0f;
            if constexpr (QT != 4) {
                // 8 bits: element e is byte e & 3 of word b (0, 1) of a k-step of lane tt, whose elements are one run of 32 in 128
#pragma unroll
                for (int j = 0; j < E / 4; ++j) {
                    uint32_t q[3] = {0, 0, 0};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x = v[4 * j + k] * inv, a = rintf(x), y = (x - a) * 254.0f, c = rintf(y), d = rintf((y - c) * 254.0f);
                        q[0] |= ((uint32_t)(int)a & 0xFFu) << (8 * k);
                        q[1] |= ((uint32_t)(int)c & 0xFFu) << (8 * k);
                        q[2] |= ((uint32_t)(int)d & 0xFFu) << (8 * k);
                    }
                    if constexpr (QT != 8) {
                        // elements 8 tt .. 8 tt + 7 of a block, as the codes lie: b0 and b1 of lane tt
                        const int e = e0 + 4 * j, half = (e >> 2) & 1, at = (row & 7) * 4 + ((e & 31) >> 3);
                        uint8_t* to = s_q + ((row >> 3) * (D / 32) + (e >> 5)) * C::QBLOCK;
                        reinterpret_cast<uint32_t*>(to)[at * 4 + half] = q[0];
                        reinterpret_cast<uint32_t*>(to)[at * 4 + 2 + half] = q[1];
                        reinterpret_cast<uint32_t*>(to + 512)[at * 2 + half] = q[2];
                        continue;
                    }
                    const int e = e0 + 4 * j, word = (e & 31) >> 2, pr = (e >> 7) * 2 + (word >> 2), tt = (e & 127) >> 5;
                    uint32_t* to = reinterpret_cast<uint32_t*>(s_q) + ((row >> 3) * (D / 64) + pr) * 384 + ((row & 7) * 4 + tt) * 4;
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        const int w = ((word >> 1) & 1) * 6 + k * 2 + (word & 1);   // of the pair of k-steps
                        to[(w >> 2) * 128 + (w & 3)] = q[k];
                    }
                }
            } else {
                // Element e of the row goes where the keys' element meets it: half-word `odd` of word w (b0, b1 of one k-step, then
                // of the next) of lane tt, pair of k-steps j2.  A pair of k-steps is a block of 32 elements, lane tt has the nibbles of
                // bytes 4 tt .. 4 tt + 3, e and e + 16 in a byte.
                __half* qh = reinterpret_cast<__half*>(s_q) + (row >> 3) * (NK / 2) * 256 + (row & 7) * 32;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const int e = e0 + j;
                    const float x = v[j] * inv;
                    const __half hi = __float2half_rn(x), lo = __float2half_rn(x - __half2float(hi));
                    const int j2 = e >> 5, tt = (e & 15) >> 2, w = e & 3;
                    const int odd = (e >> 4) & 1;
                    __half* to = qh + j2 * 256 + tt * 8 + w * 2 + odd;
                    to[0] = hi;
                    to[C::QPART / 2] = lo;
                }
            }
            if (lane == 0) {
                s_f[row] = make_float2(top * (r.sm_scale * LOG2E * C::UNIT), sees ? lse * LOG2E : INFINITY);
                s_lim[row] = sees ? last_seen(r, sl, i) : 0x7fffffff;
            }
        }
        __syncthreads();
        int lim_min = 0x7fffffff;
        if (lane < tiles * 8) lim_min = s_lim[lane];
        lim_min = __reduce_min_sync(0xffffffffu, lim_min);

        // ── blocks of 16 tokens ──
        uint32_t kt = ring - C::STAGE;
        for (int i = 0; i < mine; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
            __syncwarp();
            if ((i & 31) == 0) {
                cu_blk = nx_blk;
                cu_ks = nx_ks;
            }
            issue(i + C::STAGES - 1);
            kt += C::STAGE;
            if (kt == ring + C::RING) kt = ring;
            const int blk = __shfl_sync(0xffffffffu, cu_blk, i & 31);
            if (blk < 0) continue;                   // a page outside the pool holds nothing
            const float ks = __shfl_sync(0xffffffffu, cu_ks, i & 31);
            const int tok0 = (blk0 + warp + i * WT_WARPS) << 4, tok = tok0 + g + 8 * (t & 1);   // the token that this lane writes
            float* at = p.weights + ((int64_t)blk * 16 + (tok - tok0));

            float sum0 = 0.0f, sum1 = 0.0f;          // tokens g, g + 8, this lane's rows
            const bool edge = tok0 + 15 > lim_min;
            auto add = [&](int nt, const float (&s)[4], float ks) {
                // words 0, 1 of token g, words 2, 3 of token g + 8, for rows 2t and 2t + 1 of the tile
                const float4 f = *reinterpret_cast<const float4*>(s_f + nt * 8 + 2 * t);
                float x[4];
                x[0] = ex2(fmaf(s[0], f.x * ks, -f.y));
                x[1] = ex2(fmaf(s[1], f.z * ks, -f.w));
                x[2] = ex2(fmaf(s[2], f.x * ks, -f.y));
                x[3] = ex2(fmaf(s[3], f.z * ks, -f.w));
                if (edge) {
                    asm volatile("" ::: "memory");   // the last blocks only: kept a branch
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int left = s_lim[nt * 8 + 2 * t + e] - tok0 - g;
                        if (left < 0) x[e] = 0.0f;
                        if (left < 8) x[2 + e] = 0.0f;
                    }
                }
                sum0 += x[0] + x[1];
                sum1 += x[2] + x[3];
            };
            if constexpr (QT == 8) {
                uint32_t a[D / 32][4];
#pragma unroll
                for (int half = 0; half < D / 128; ++half)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t row = kt + half * 2048 + (x * 8 + g) * 128;
                        const uint4 u = wt_lds128(row + (((2 * t) ^ g) << 4)), w = wt_lds128(row + (((2 * t + 1) ^ g) << 4));
                        a[half * 4][x] = u.x; a[half * 4][2 + x] = u.y; a[half * 4 + 1][x] = u.z; a[half * 4 + 1][2 + x] = u.w;
                        a[half * 4 + 2][x] = w.x; a[half * 4 + 2][2 + x] = w.y; a[half * 4 + 3][x] = w.z; a[half * 4 + 3][2 + x] = w.w;
                    }
                for (int nt = 0; nt < tiles; ++nt) {
                    int c[3][4];
#pragma unroll
                    for (int k = 0; k < 3; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[k][e] = 0x4B400000;   // 1.5 * 2^23
#pragma unroll
                    for (int pr = 0; pr < D / 64; ++pr) {
                        const uint32_t from = sq + (nt * (D / 64) + pr) * 1536;
                        const uint4 u = wt_lds128(from), v = wt_lds128(from + 512), w = wt_lds128(from + 1024);
                        wt_imma(c[0], a[2 * pr], u.x, u.y);
                        wt_imma(c[1], a[2 * pr], u.z, u.w);
                        wt_imma(c[2], a[2 * pr], v.x, v.y);
                        wt_imma(c[0], a[2 * pr + 1], v.z, v.w);
                        wt_imma(c[1], a[2 * pr + 1], w.x, w.y);
                        wt_imma(c[2], a[2 * pr + 1], w.z, w.w);
                    }
                    float s[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        constexpr float ZERO = 12582912.0f;
                        s[e] = fmaf(__int_as_float(c[2][e]) - ZERO, 1.0f / (254.0f * 254.0f), (__int_as_float(c[1][e]) - ZERO) * (1.0f / 254.0f));
                        s[e] += __int_as_float(c[0][e]) - ZERO;
                    }
                    add(nt, s, ks);
                }
            } else if constexpr (QT != 4) {
                // A block of 32 elements is a k-step; a lane takes the 8 codes of elements 8 t .. 8 t + 7 of tokens g and g + 8.  Codes
                // become the nibbles of a byte permute's selector, which looks up four levels' terms at a time.
                constexpr int BB = BlockBytes<QT>::value;
                constexpr float Z = 12582912.0f, R2 = 1.0f / (254.0f * 254.0f);
                float2 acc[TILES][2];
#pragma unroll
                for (int nt = 0; nt < TILES; ++nt) acc[nt][0] = acc[nt][1] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j2 = 0; j2 < D / 32; ++j2) {
                    float d[2];
                    uint32_t a[3][4];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t row = kt + (x * 8 + g) * C::ROWB + j2 * BB;
                        d[x] = scale_decode(wt_lds16s(row));
                        uint32_t v;
                        if constexpr (QT == 3) {
                            // bytes 3 t .. 3 t + 2 of the codes: two half-words, from byte 3 t or the one before
                            const uint32_t from = row + 2 + ((3 * t) & ~1);
                            v = wt_prmt(wt_lds16(from), wt_lds16(from + 2), (t & 1) ? 0x5541u : 0x5410u);
                            v = wt_either(0x0000FFFFu, v, v << 4);   // 12 bits in 16
                            v = wt_either(0x00FF00FFu, v, v << 2);   // 6 in 8
                            v = (v & 0x07070707u) | ((v << 1) & 0x70707070u);
                        } else {
                            const uint32_t w = wt_lds16(row + 2 + 2 * t);
                            v = wt_either(0x0000FFFFu, w, w << 8);
                            v = wt_either(0x00FF00FFu, v, v << 4);
                            v = (v & 0x03030303u) | ((v << 2) & 0x30303030u);
                        }
#pragma unroll
                        for (int k = 0; k < 3; ++k) {
                            a[k][x] = wt_prmt(levels[k][0], levels[k][1], v);
                            a[k][2 + x] = wt_prmt(levels[k][0], levels[k][1], v >> 16);
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < TILES; ++nt) {
                        if (nt >= tiles) break;
                        const uint32_t from = (uint32_t)__cvta_generic_to_shared(s_q) + (nt * (D / 32) + j2) * C::QBLOCK;
                        const uint4 q = wt_lds128(from + lane * 16);
                        const uint2 q3 = wt_lds64(from + 512 + lane8);
                        // products by the size of their terms; those below 2^-23 of the largest elements are left out
                        int c[3][4];
                        wt_imma_first(c[0], a[0], q.x, q.y, 0x4B400000);
                        wt_imma_first(c[1], a[0], q.z, q.w, 0x4B400000);
                        wt_imma_first(c[2], a[0], q3.x, q3.y, 0x4B400000);
                        wt_imma(c[1], a[1], q.x, q.y);
                        wt_imma(c[2], a[1], q.z, q.w);
                        wt_imma(c[2], a[2], q.x, q.y);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const auto pair = [&](int k) { return make_float2(__int_as_float(c[k][2 * x]), __int_as_float(c[k][2 * x + 1])); };
                            // -Z R2 is rounded by 2^-17 of the first term's unit
                            float2 y = __ffma2_rn(pair(2), make_float2(R2, R2), make_float2(-Z * R2, -Z * R2));
                            y = __ffma2_rn(__fadd2_rn(pair(1), make_float2(-Z, -Z)), make_float2(1.0f / 254.0f, 1.0f / 254.0f), y);
                            y = __fadd2_rn(y, __fadd2_rn(pair(0), make_float2(-Z, -Z)));
                            acc[nt][x] = __ffma2_rn(y, make_float2(d[x], d[x]), acc[nt][x]);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < TILES; ++nt) {
                    const float y[4] = {acc[nt][0].x, acc[nt][0].y, acc[nt][1].x, acc[nt][1].y};
                    if (nt < tiles) add(nt, y, 1.0f);
                }
            } else {
                // a block of 32 elements is two k-steps; its scales are those of tokens g and g + 8
                float acc[TILES][4];
#pragma unroll
                for (int nt = 0; nt < TILES; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
                constexpr int BB = BlockBytes<QT>::value;
#pragma unroll
                for (int j2 = 0; j2 < D / 32; ++j2) {
                    float d[2];
                    uint2 lv[2][4];   // two f16 terms of the pairs of levels, tokens g and g + 8
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t row = kt + (x * 8 + g) * C::ROWB + j2 * BB;
                        d[x] = scale_decode(wt_lds16s(row));
                        uint32_t at[4];   // of the pairs in the table
                        const uint32_t w = wt_lds16(row + 2 + 4 * t) | wt_lds16(row + 4 + 4 * t) << 16;
#pragma unroll
                        for (int i4 = 0; i4 < 4; ++i4) at[i4] = __byte_perm(w, lane8, 0x5504 | i4 << 4);   // lane8 is below 256
#pragma unroll
                        for (int i4 = 0; i4 < 4; ++i4) lv[x][i4] = *reinterpret_cast<const uint2*>(smem + at[i4]);
                    }
                    // A product takes 8 tokens: the first terms of their levels in its rows 0 .. 7, the second ones in rows 8 .. 15, as
                    // the lookups give them (16 tokens a product and a product for each term would be 6 of them instead of 8,
                    // and 16 moves of registers)
#pragma unroll
                    for (int nt = 0; nt < TILES; ++nt) {
                        if (nt >= tiles) break;
                        const uint32_t from = sq + (nt * (NK / 2) + j2) * 512;
                        const uint4 q = wt_lds128(from), ql = wt_lds128(from + C::QPART);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t a0[4] = {lv[x][0].x, lv[x][0].y, lv[x][1].x, lv[x][1].y};
                            const uint32_t a1[4] = {lv[x][2].x, lv[x][2].y, lv[x][3].x, lv[x][3].y};
                            float s[4];
                            wt_mma_first(s, a0, q.x, q.y);
                            wt_mma(s, a1, q.z, q.w);
                            wt_mma(s, a0, ql.x, ql.y);
                            wt_mma(s, a1, ql.z, ql.w);
                            acc[nt][2 * x] = fmaf(s[0] + s[2], d[x], acc[nt][2 * x]);
                            acc[nt][2 * x + 1] = fmaf(s[1] + s[3], d[x], acc[nt][2 * x + 1]);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < TILES; ++nt)
                    if (nt < tiles) add(nt, acc[nt], 1.0f);
            }
            // the rows of the four lanes
            sum0 += __shfl_xor_sync(0xffffffffu, sum0, 1);
            sum1 += __shfl_xor_sync(0xffffffffu, sum1, 1);
            sum0 += __shfl_xor_sync(0xffffffffu, sum0, 2);
            sum1 += __shfl_xor_sync(0xffffffffu, sum1, 2);
            if (t < 2 && tok < end) {
                float x = t ? sum1 : sum0;
                if (chunk > 0) x += s_sum[tok - begin];
                if (reads && tok < fresh) x = fmaf(p.decay, wt_lds32(kt + C::TILE + (tok - tok0) * 4), x);
                if (last) *at = x;
                else s_sum[tok - begin] = x;
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (last) break;
    }
    }
}

WeightsPlan weights_plan(int B, int Hkv, int grp, int D, int64_t n, int64_t max_len, bool q8) {
    WeightsPlan p;
    const int64_t rows = n * grp, len = max_len > 0 ? max_len : 1, pairs = (int64_t)B * Hkv;
    p.pairs_pass = (int)pairs;
    p.tensor = q8 && rows > WT_ROWS;   // both sides measured: the table above
    if (p.tensor) {
        weights_rows_plan(pairs, D, rows, len, &p);
        return p;
    }
    p.rows = rows <= 8 ? 8 : WT_ROWS;
    p.chunks = (int)((rows + p.rows - 1) / p.rows);
    if (p.chunks < 1) p.chunks = 1;
    const int64_t slots = 3 * (int64_t)sm_count();
    // A CTA's time is its tokens plus a start worth some.  Sequences differ in length, and the grid is made for the longest:
    // rather several waves of short CTAs than one of long ones, as far as the start lets them.
    int64_t best = INT64_MAX;
    for (int s = 1; s <= 256; ++s) {
        const int64_t per = ((len + s - 1) / s + 127) / 128 * 128;
        if (s > 1 && (int64_t)(s - 1) * per >= len) continue;
        const int64_t waves = (pairs * s + slots - 1) / slots, cost = waves * (per + WT_START) + per;
        if (cost < best) { best = cost; p.splits = s; }
        if (waves > 16) break;
    }
    return p;
}

template <int D, int QT, int TILES> static cudaError_t launch_weights_t(const WeightsRun& r, const WeightsPlan& p, cudaStream_t st) {
    using C = WtCfg<D, QT, TILES>;
    const cudaError_t e = allow_smem(weights_kernel<D, QT, TILES>, C::SMEM);
    if (e != cudaSuccess) return e;
    const int64_t grid = (int64_t)r.q.B * r.q.Hkv * p.splits;
    if (grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    weights_kernel<D, QT, TILES><<<(unsigned)grid, WT_THREADS, C::SMEM, st>>>(r, p.splits, p.chunks);
    return cudaGetLastError();
}

cudaError_t launch_weights(const WeightsRun& r, const WeightsPlan& p, void* workspace, cudaStream_t st) {
    if (p.tensor) return launch_weights_rows(r, p, workspace, st);
    const auto run = [&](auto d) {
        constexpr int D = decltype(d)::value;
        switch (r.k_type) {
            case 8: return p.rows == 8 ? launch_weights_t<D, 8, 1>(r, p, st) : launch_weights_t<D, 8, 4>(r, p, st);
            case 4: return p.rows == 8 ? launch_weights_t<D, 4, 1>(r, p, st) : launch_weights_t<D, 4, 4>(r, p, st);
            case 3: return p.rows == 8 ? launch_weights_t<D, 3, 1>(r, p, st) : launch_weights_t<D, 3, 4>(r, p, st);
            default: return p.rows == 8 ? launch_weights_t<D, 2, 1>(r, p, st) : launch_weights_t<D, 2, 4>(r, p, st);
        }
    };
    return r.q.D == 256 ? run(std::integral_constant<int, 256>()) : run(std::integral_constant<int, 128>());
}

}  // namespace tq
