// tq_rope.cu — rotation of head rows by position, alone and fused into the paged append.
//
// Kernels
//   rotary_kernel<T>                  queries and keys rotated (or rotated back) into strided outputs
//   rotary_append_kernel<D, T, KT>    keys: rotate by position, Hadamard, quantize into pages; values: Hadamard,
//                                     quantize into pages; queries: rotate.  One launch for all three.
//   dequantize_q8_kernel<T>           values of 8-bit pages
//
// Angles.  A pair turns by p * f with p an integer position, so only the fraction of p * f / 2 pi matters.
// F = floor(f / (2 pi) * 2^64) is within 2^-64 of a turn, and p * F mod 2^64 is that fraction within p 2^-64
// (3e-13 radians at a million positions; nothing is lost to p itself).  The fraction is folded to an eighth of a turn and its sine and cosine are Taylor
// sums in 64 bits (the next term is below 2^-54), rounded once to 32 bits: the same values as 64-bit library
// functions rounded to 32 bits give, at any position, so quantized codes do not depend on who computed the
// angle.  They cost about 60 instructions for a pair; a CTA takes 16 tokens and keeps their angles in shared
// memory for all its heads.
//
// Bit-exactness: rotation, Hadamard stages and quantization are single fp32 operations, each correctly
// rounded, in the order of the separate operations (x c - y s with three roundings, stages h = 1, 2, 4, ...).
#include <type_traits>

#include "tq_common.cuh"
#include "tq_kernels.h"
#include "tq_rope.h"
#include "tq_rows.cuh"

namespace tq {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_WARPS = ROPE_THREADS / 32;
constexpr int ROPE_TOKENS = 16;   // tokens per CTA, and slots per 8-bit scale block

// ── angles ─────────────────────────────────────────────────────────────────

// floor(2^130 / (2 pi)) = floor(2^129 / pi): the 128 leading bits of 1 / (2 pi)
constexpr uint64_t INV_2PI_HI = 0xA2F9836E4E441529ull, INV_2PI_LO = 0xFC2757D1F534DDC0ull;

// f / (2 pi) * 2^64 mod 2^64.  f = m 2^e with a 53-bit m; m * (2^130 / 2 pi) has up to 181 bits, of which the
// result is those from 66 - e on (e below -115 gives 0; |f| >= 2^31 and non-finite f are taken as 0).
__device__ __forceinline__ uint64_t turn_fraction(double f) {
    const uint64_t u = (uint64_t)__double_as_longlong(f);
    const int ex = (int)((u >> 52) & 0x7FF);
    const int e = ex - 1075;
    if (ex == 0 || e > -22) return 0;
    const uint64_t m = (u & 0xFFFFFFFFFFFFFull) | (1ull << 52);
    const uint64_t w0 = m * INV_2PI_LO, c0 = __umul64hi(m, INV_2PI_LO);
    const uint64_t w1 = m * INV_2PI_HI + c0;
    const uint64_t w2 = __umul64hi(m, INV_2PI_HI) + (w1 < c0 ? 1 : 0);
    const int s = 66 - e;          // >= 88
    uint64_t r;
    if (s < 128) r = (w1 >> (s - 64)) | (w2 << (128 - s));
    else if (s < 192) r = w2 >> (s - 128);
    else r = 0;
    (void)w0;
    return (u >> 63) ? 0 - r : r;
}

// cosine and sine of fraction / 2^64 turns, times scale, rounded to fp32
__device__ __forceinline__ float2 turn_cos_sin(uint64_t fraction, double scale) {
    const uint64_t q = (fraction + (1ull << 61)) >> 62;             // nearest quarter turn
    const int64_t r = (int64_t)(fraction - (q << 62));              // within an eighth of a turn of it
    const double x = (double)r * 3.4061215800865545e-19;            // 2 pi / 2^64
    const double z = x * x;
    double s = -1.0 / 1307674368000.0;                              // -1 / 15!
    s = fma(s, z, 1.0 / 6227020800.0);
    s = fma(s, z, -1.0 / 39916800.0);
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, x, x);
    double c = 1.0 / 20922789888000.0;                              // 1 / 16!
    c = fma(c, z, -1.0 / 87178291200.0);
    c = fma(c, z, 1.0 / 479001600.0);
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const double cq = (q & 1) ? -s : c, sq = (q & 1) ? c : s;       // quarter turns 0 .. 3 (q mod 4)
    const double sg = (q & 2) ? -scale : scale;
    return make_float2((float)(cq * sg), (float)(sq * sg));
}

// Shared angle table of 16 tokens: pair i of token row r is the (cos, sin) half (i & 1) of the 16-byte entry
// (r, (i >> 1) & 3, i >> 3): the lanes of a row, which read whole runs of 8 pairs, read consecutive entries.
__device__ __forceinline__ int angle_at(int row, int pair, int n8) {
    return (((row * 4 + ((pair >> 1) & 3)) * n8 + (pair >> 3)) << 1) + (pair & 1);
}

// angles of the CTA's tokens: row r is token t0 + r of sequence b (rows outside [0, n_new) are left out)
__device__ __forceinline__ void fill_angles(float2* __restrict__ tab, const Rope& rope, int b, int batch, int64_t t0,
                                            int64_t n_new, int64_t first) {
    const int pairs = rope.rotary_dim >> 1, n8 = (pairs + 7) >> 3;
    const int per = ROPE_THREADS / pairs;                           // rows per sweep; pairs <= ROPE_THREADS
    const int row0 = threadIdx.x / pairs;
    if (row0 >= per) return;
    const int pair = threadIdx.x - row0 * pairs;
    const uint64_t step = turn_fraction(rope.inv_freq[pair]);
    int ax = rope.axis ? rope.axis[pair] : 0;
    ax = ax < 0 ? 0 : (ax >= rope.n_axes ? rope.n_axes - 1 : ax);   // device data: kept inside the positions
    for (int row = row0; row < ROPE_TOKENS; row += per) {
        const int64_t t = t0 + row;
        if (t < 0 || t >= n_new) continue;
        const int64_t p = rope.positions ? (int64_t)rope.positions[((int64_t)ax * batch + b) * n_new + t] : first + t;
        float2 cs = turn_cos_sin((uint64_t)p * step, rope.scale);
        if (rope.inverse) cs.y = -cs.y;
        tab[angle_at(row, pair, n8)] = cs;
    }
}

// ── rows ───────────────────────────────────────────────────────────────────

// the 8 angles of pairs 8 c .. 8 c + 7 of a token row
__device__ __forceinline__ void angles8(const float2* __restrict__ tab, int row, int c, int n8, float (&cs)[8],
                                        float (&sn)[8]) {
    const float4* e = reinterpret_cast<const float4*>(tab) + row * 4 * n8 + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float4 w = e[j * n8];
        cs[2 * j] = w.x; sn[2 * j] = w.y; cs[2 * j + 1] = w.z; sn[2 * j + 1] = w.w;
    }
}
// the 4 angles of pairs 4 c .. 4 c + 3 (8 neighbouring elements of interleaved pairs)
__device__ __forceinline__ void angles4(const float2* __restrict__ tab, int row, int c, int n8, float (&cs)[4],
                                        float (&sn)[4]) {
    const float4* e = reinterpret_cast<const float4*>(tab) + (row * 4 + 2 * (c & 1)) * n8 + (c >> 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float4 w = e[j * n8];
        cs[2 * j] = w.x; sn[2 * j] = w.y; cs[2 * j + 1] = w.z; sn[2 * j + 1] = w.w;
    }
}
__device__ __forceinline__ float rot_lo(float a, float b, float c, float s) {
    return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}
__device__ __forceinline__ float rot_hi(float a, float b, float c, float s) {
    return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}
__device__ __forceinline__ void turn_neighbours(float (&v)[8], const float2* __restrict__ tab, int row, int c, int n8) {
    float cs[4], sn[4];
    angles4(tab, row, c, n8, cs, sn);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = v[2 * j], b = v[2 * j + 1];
        v[2 * j] = rot_lo(a, b, cs[j], sn[j]);
        v[2 * j + 1] = rot_hi(a, b, cs[j], sn[j]);
    }
}

// Rotates token rows [r0, r1) of one head: an item is one row's pair of 8-element runs that turn into each
// other (c and c + R / 16 runs on), or two runs that are only copied.  Every element is read and written by
// one thread, so dst may be src.
template <typename T>
__device__ __forceinline__ void rope_rows(const T* __restrict__ src, int64_t src_tok, T* dst, int64_t dst_tok, int D,
                                          const Rope& rope, const float2* __restrict__ tab, int64_t t0, int r0, int r1,
                                          int lane, int lanes) {
    const int R = rope.rotary_dim, n8 = ((R >> 1) + 7) >> 3, half8 = R >> 4;
    const int per = (D + 15) >> 4;   // items per row
    for (int it = lane; it < (r1 - r0) * per; it += lanes) {
        const int row = r0 + it / per, c = it % per;
        const T* s = src + (t0 + row) * src_tok;
        T* d = dst + (t0 + row) * dst_tok;
        float a[8], b[8];
        if (c < half8 && !rope.interleaved) {
            load8<T>(s + 8 * c, a);
            load8<T>(s + 8 * c + (R >> 1), b);
            float cs[8], sn[8];
            angles8(tab, row, c, n8, cs, sn);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = a[j], y = b[j];
                a[j] = rot_lo(x, y, cs[j], sn[j]);
                b[j] = rot_hi(x, y, cs[j], sn[j]);
            }
            store8<T>(d + 8 * c, a);
            store8<T>(d + 8 * c + (R >> 1), b);
        } else if (c < half8) {
            load8<T>(s + 16 * c, a);
            load8<T>(s + 16 * c + 8, b);
            turn_neighbours(a, tab, row, 2 * c, n8);
            turn_neighbours(b, tab, row, 2 * c + 1, n8);
            store8<T>(d + 16 * c, a);
            store8<T>(d + 16 * c + 8, b);
        } else if (s != d) {
            load8<T>(s + 16 * c, a);
            store8<T>(d + 16 * c, a);
            if (16 * c + 8 < D) {
                load8<T>(s + 16 * c + 8, b);
                store8<T>(d + 16 * c + 8, b);
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(ROPE_THREADS) rotary_kernel(const RotaryRun r, int tiles, int groups, int per_group) {
    extern __shared__ __align__(16) uint8_t smem[];
    float2* tab = reinterpret_cast<float2*>(smem);
    const int g = blockIdx.x % groups, tile = (blockIdx.x / groups) % tiles, b = blockIdx.x / groups / tiles;
    const int64_t t0 = (int64_t)tile * ROPE_TOKENS;
    const int rows = (int)(r.n_new - t0 < ROPE_TOKENS ? r.n_new - t0 : ROPE_TOKENS);
    fill_angles(tab, r.rope, b, r.batch, t0, r.n_new, 0);
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h0 = r.x[0].heads, total = h0 + r.x[1].heads;
    const int end = (g + 1) * per_group < total ? (g + 1) * per_group : total;
    for (int u = g * per_group + warp; u < end; u += ROPE_WARPS) {
        const HeadRows& x = r.x[u >= h0];
        const int h = u >= h0 ? u - h0 : u;
        rope_rows<T>(static_cast<const T*>(x.src) + b * x.ss[0] + h * x.ss[1], x.ss[2],
                     static_cast<T*>(x.dst) + b * x.ds[0] + h * x.ds[1], x.ds[2], r.head_dim, r.rope, tab, t0, 0, rows,
                     lane, 32);
    }
}

// ── append ─────────────────────────────────────────────────────────────────

// elements e .. e + 7 of a key row, turned: the partners are read from the row again (they sit in the L1)
template <typename T>
__device__ __forceinline__ void turned8(const T* __restrict__ row_ptr, int e, const Rope& rope,
                                        const float2* __restrict__ tab, int row, int n8, float (&v)[8]) {
    load8<T>(row_ptr + e, v);
    const int R = rope.rotary_dim;
    if (e >= R) return;
    if (rope.interleaved) {
        turn_neighbours(v, tab, row, e >> 3, n8);
        return;
    }
    const int hi = e >= (R >> 1);
    const int c = (hi ? e - (R >> 1) : e) >> 3;
    float p[8], cs[8], sn[8];
    load8<T>(row_ptr + (hi ? e - (R >> 1) : e + (R >> 1)), p);
    angles8(tab, row, c, n8, cs, sn);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = hi ? rot_hi(p[j], v[j], cs[j], sn[j]) : rot_lo(v[j], p[j], cs[j], sn[j]);
}

// Packs the 16 codes of a lane (half `odd` of a 32-element block) into the staged block at blk.
template <int QT>
__device__ __forceinline__ void stage_half_block(uint8_t* __restrict__ blk, const uint32_t (&code)[16], int odd,
                                                 uint16_t d) {
    if (!odd) *reinterpret_cast<uint16_t*>(blk) = d;
    if constexpr (QT == 4) {   // byte j = code j | code j + 16 << 4: the even lane packs bytes 0..7, the odd 8..15
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo |= code[j] << (4 * j);
            hi |= code[8 + j] << (4 * j);
        }
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? lo : hi, 1);
        const uint32_t a = odd ? other : lo, b = odd ? hi : other;   // nibbles of elements j and j + 16
        uint16_t* w = reinterpret_cast<uint16_t*>(blk + 2 + 8 * odd);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = (a >> (8 * i)) & 0xFFu, y = (b >> (8 * i)) & 0xFFu;
            w[i] = (uint16_t)((x & 15u) | ((y & 15u) << 4) | ((x >> 4) << 8) | ((y >> 4) << 12));
        }
    } else if constexpr (QT == 3) {   // two 24-bit groups of 8 codes
        uint32_t g[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[0] |= code[j] << (3 * j);
            g[1] |= code[8 + j] << (3 * j);
        }
        uint16_t* w = reinterpret_cast<uint16_t*>(blk + 2 + 6 * odd);
        w[0] = (uint16_t)g[0];
        w[1] = (uint16_t)((g[0] >> 16) | (g[1] << 8));
        w[2] = (uint16_t)(g[1] >> 8);
    } else {
        uint32_t g = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) g |= code[j] << (2 * j);
        uint16_t* w = reinterpret_cast<uint16_t*>(blk + 2 + 4 * odd);
        w[0] = (uint16_t)g;
        w[1] = (uint16_t)(g >> 16);
    }
}

// where a 16-slot tile of one (sequence, head) lies: offset in rows, or -1 (outside the cache or the pool)
__device__ __forceinline__ int64_t tile_rows_at(const RotaryAppendRun& r, int b, int h, int64_t slot0) {
    if (slot0 < 0 || slot0 >= (r.max_pages << r.page_shift)) return -1;
    const int32_t pg = r.pages[(int64_t)b * r.max_pages + (slot0 >> r.page_shift)];
    if (pg < 0 || pg >= r.num_pages) return -1;
    return ((((int64_t)pg * r.n_kv_heads + h) << r.page_shift) + (slot0 & ((int64_t(1) << r.page_shift) - 1)));
}

constexpr int STAGE_BYTES = 16 * 72;   // packed rows that a warp stages: 16 of D = 128 or 8 of D = 256

// One (sequence, K or V head, 16-slot tile): rows [ra, rb) of the tile are new.  D / 128 warps take a unit,
// `sub` the warp's index among them; each holds 16 elements of 16 * 32 / D rows at a time.
template <int D, typename T, int QT>
__device__ __forceinline__ void append_unit(const RotaryAppendRun& r, const HeadRows& x, const PoolDst& dst, bool turn,
                                            int b, int h, int64_t slot0, int64_t t0, int ra, int rb, int older,
                                            const float2* __restrict__ tab, uint8_t* __restrict__ stage,
                                            float* __restrict__ s_amax, int sub, int bar) {
    constexpr int LPR = D / 16, RPP = 32 / LPR, WPU = D / 128, RPW = 16 / WPU, PASSES = RPW / RPP;
    const int lane = threadIdx.x & 31, lr = lane / LPR, le = (lane % LPR) * 16;
    const int64_t at = tile_rows_at(r, b, h, slot0);
    if (at < 0) {
        if (r.overflow && lane == 0 && sub == 0) atomicAdd(r.overflow, rb - ra);
        return;
    }
    const T* src = static_cast<const T*>(x.src) + b * x.ss[0] + h * x.ss[1] + t0 * x.ss[2];
    const int n8 = ((r.rope.rotary_dim >> 1) + 7) >> 3;

    auto row_values = [&](int row, float (&v)[16]) {
        float a[8], c[8];
        if (row >= ra && row < rb) {
            const T* p = src + row * x.ss[2];
            if (turn) {
                turned8<T>(p, le, r.rope, tab, row, n8, a);
                turned8<T>(p, le + 8, r.rope, tab, row, n8, c);
            } else {
                load8<T>(p + le, a);
                load8<T>(p + le + 8, c);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) { v[j] = a[j]; v[8 + j] = c[j]; }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.0f;
        }
        if (r.rotate) fwht16<D>(v, r.norm);
    };

    if constexpr (QT == 8) {
        float v[PASSES][16];
        float amax = 0.0f;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int base = sub * RPW + p * RPP;
            if (base + RPP <= ra || base >= rb) {   // no new row in this pass (the same for all lanes)
#pragma unroll
                for (int j = 0; j < 16; ++j) v[p][j] = 0.0f;
                continue;
            }
            row_values(base + lr, v[p]);
#pragma unroll
            for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(v[p][j]));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        float* sp = dst.scale + (at >> 4);
        const float s_old = older > 0 ? *sp : 0.0f;
        if constexpr (WPU == 2) {
            // the two warps of the unit exchange their maxima; the old scale has been read by both
            if (lane == 0) s_amax[sub] = amax;
            asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
            amax = fmaxf(s_amax[0], s_amax[1]);
            asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
        }
        // A block's scale only grows while the block fills, so codes written earlier stay in range; it starts
        // anew with slot 0.  Scales below 2^-100 (all values below 1e-28) are stored as zero.
        float s = fmaxf(s_old, __fmul_rn(amax, 1.0f / 127.0f));
        if (!(s >= 0x1p-100f)) s = 0.0f;
        const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
        int8_t* pool = reinterpret_cast<int8_t*>(dst.pool) + at * D;
        const bool grow = older > 0 && s_old < s;
        const float ratio = __fmul_rn(s_old, inv);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int row = sub * RPW + p * RPP + lr;
            uint4* cell = reinterpret_cast<uint4*>(pool + row * D + le);
            if (row >= ra && row < rb) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t acc = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        int c = __float2int_rn(__fmul_rn(v[p][4 * i + j], inv));
                        c = c < -127 ? -127 : (c > 127 ? 127 : c);
                        acc |= (uint32_t)(c & 0xFF) << (8 * j);
                    }
                    w[i] = acc;
                }
                *cell = make_uint4(w[0], w[1], w[2], w[3]);
            } else if (grow && row < older) {
                const uint4 o = *cell;
                const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t acc = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int c = (int)(int8_t)(ow[i] >> (8 * j));
                        acc |= (uint32_t)(__float2int_rn(__fmul_rn((float)c, ratio)) & 0xFF) << (8 * j);
                    }
                    w[i] = acc;
                }
                *cell = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        if (lane == 0 && sub == 0 && s != s_old) *sp = s;
        else if (lane == 0 && sub == 0 && older == 0) *sp = s;
    } else {
        constexpr int BB = BlockBytes<QT>::value, ROWB = D / 32 * BB;
#pragma unroll 1
        for (int p = 0; p < PASSES; ++p) {
            const int base = sub * RPW + p * RPP, row = base + lr;
            if (base + RPP <= ra || base >= rb) continue;
            float v[16];
            row_values(row, v);
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(v[j]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            const float inv = amax > 0.0f ? __fdiv_rn(1.0f, amax) : 0.0f;
            uint32_t code[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float xn = __fmul_rn(v[j], inv);
                code[j] = (uint32_t)(QT == 4 ? tq4_nearest(xn) : QT == 3 ? tq3_nearest(xn) : tq2_nearest(xn));
            }
            stage_half_block<QT>(stage + (row - sub * RPW) * ROWB + (le >> 5) * BB, code, (le >> 4) & 1, half_trunc(amax));
        }
        __syncwarp();
        // the new rows are consecutive slots of one page: one run of 8-byte words
        const int lo = ra > sub * RPW ? ra : sub * RPW, hi = rb < (sub + 1) * RPW ? rb : (sub + 1) * RPW;
        const uint2* from = reinterpret_cast<const uint2*>(stage + (lo - sub * RPW) * ROWB);
        uint2* to = reinterpret_cast<uint2*>(dst.pool + (at + lo) * ROWB);
        for (int i = lane; i < (hi - lo) * (ROWB / 8); i += 32) to[i] = from[i];
        __syncwarp();
    }
}

// Work of a CTA: 16 slot-aligned tokens of one sequence, heads [g * per_group, ...) of the list
// K heads | V heads | query heads.  The slot alignment gives an 8-bit scale block to one unit.
template <int D, typename T, int KT>
__global__ void __launch_bounds__(ROPE_THREADS, 2)
rotary_append_kernel(const RotaryAppendRun r, int tiles, int groups, int per_group) {
    constexpr int WPU = D / 128, VT = KT == 8 ? 8 : 4;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(16) uint8_t s_stage[KT == 8 ? 16 : ROPE_WARPS * STAGE_BYTES];
    __shared__ float s_amax[ROPE_WARPS];
    float2* tab = reinterpret_cast<float2*>(smem);
    const int g = blockIdx.x % groups, tile = (blockIdx.x / groups) % tiles, b = blockIdx.x / groups / tiles;
    const int64_t pos = r.pos ? r.pos[b] : 0;
    const int64_t slot0 = ((pos >> 4) + tile) << 4, t0 = slot0 - pos;   // t0 in (-16, ...)
    if (t0 >= r.n_new) return;
    int64_t len = r.new_len ? r.new_len[b] : r.n_new;
    len = len < 0 ? 0 : (len > r.n_new ? r.n_new : len);
    const bool turn = r.rope.inv_freq != nullptr;
    if (turn) {
        fill_angles(tab, r.rope, b, r.batch, t0, r.n_new, pos);
        __syncthreads();
    }
    const int ra = t0 < 0 ? (int)-t0 : 0;
    const int rb = len - t0 < ROPE_TOKENS ? (int)(len - t0) : ROPE_TOKENS;        // stored rows of the tile
    const int rq = r.n_new - t0 < ROPE_TOKENS ? (int)(r.n_new - t0) : ROPE_TOKENS;   // query rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WPU;
    const int Hkv = r.n_kv_heads, total = 2 * Hkv + r.q.heads;
    const int end = (g + 1) * per_group < total ? (g + 1) * per_group : total;
    for (int u = g * per_group + warp / WPU; u < end; u += ROPE_WARPS / WPU) {
        uint8_t* stage = s_stage + (KT == 8 ? 0 : warp * STAGE_BYTES);
        float* am = s_amax + (warp - sub);
        const int bar = 1 + warp / WPU;
        if (u < Hkv) {
            if (ra < rb) append_unit<D, T, KT>(r, r.k, r.kd, turn, b, u, slot0, t0, ra, rb, ra, tab, stage, am, sub, bar);
        } else if (u < 2 * Hkv) {
            if (ra < rb) append_unit<D, T, VT>(r, r.v, r.vd, false, b, u - Hkv, slot0, t0, ra, rb, ra, tab, stage, am, sub, bar);
        } else {
            const int h = u - 2 * Hkv;
            rope_rows<T>(static_cast<const T*>(r.q.src) + b * r.q.ss[0] + h * r.q.ss[1], r.q.ss[2],
                         static_cast<T*>(r.q.dst) + b * r.q.ds[0] + h * r.q.ds[1], r.q.ds[2], D, r.rope, tab, t0, ra, rq,
                         lane + 32 * sub, 32 * WPU);
        }
    }
}

// ── 8-bit pages to values ──────────────────────────────────────────────────
// a thread decodes 16 codes (one 16-byte load)
template <typename T>
__global__ void __launch_bounds__(256) dequantize_q8_kernel(const uint4* __restrict__ code, const float* __restrict__ scale,
                                                            T* __restrict__ y, int64_t n16, int log2_per_block) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256) {
        const uint4 w = code[i];
        const float s = scale[i >> log2_per_block];
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        float v[2][8];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j >> 3][j & 7] = __fmul_rn((float)(int)(int8_t)(u[j >> 2] >> (8 * (j & 3))), s);
        store8<T>(y + 16 * i, v[0]);
        store8<T>(y + 16 * i + 8, v[1]);
    }
}

// ── launches ───────────────────────────────────────────────────────────────

// Heads per CTA.  One CTA for all heads of a tile computes the tile's angles once; a batch of few tokens
// spreads its heads over CTAs instead (down to one unit per warp) until the grid covers the SMs twice.
static void split_heads(int64_t tiles, int total, int slots, int& groups, int& per_group) {
    const int64_t want = 2 * (int64_t)sm_count();
    int64_t g = (want + tiles - 1) / tiles;
    const int most = (total + slots - 1) / slots;
    if (g > most) g = most;
    if (g < 1) g = 1;
    per_group = (int)((total + g - 1) / g);
    per_group = (per_group + slots - 1) / slots * slots;
    groups = (total + per_group - 1) / per_group;
}

static size_t angle_bytes(const Rope& r) {
    return r.inv_freq ? (size_t)ROPE_TOKENS * 4 * ((r.rotary_dim / 2 + 7) / 8) * 16 : 0;
}

cudaError_t launch_rotary(const RotaryRun& r, cudaStream_t st) {
    const int64_t tiles = (r.n_new + ROPE_TOKENS - 1) / ROPE_TOKENS;
    int groups, per;
    split_heads(tiles * r.batch, r.x[0].heads + r.x[1].heads, ROPE_WARPS, groups, per);
    const int64_t grid = tiles * r.batch * groups;
    if (grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    const size_t sm = angle_bytes(r.rope);
    if (r.dtype == DT_F32) rotary_kernel<float><<<(unsigned)grid, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per);
    else if (r.dtype == DT_F16) rotary_kernel<__half><<<(unsigned)grid, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per);
    else rotary_kernel<__nv_bfloat16><<<(unsigned)grid, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per);
    return cudaGetLastError();
}

template <int D, typename T>
static cudaError_t launch_append(const RotaryAppendRun& r, cudaStream_t st) {
    const int64_t tiles = (r.n_new + 2 * ROPE_TOKENS - 2) / ROPE_TOKENS;   // any alignment of the first slot
    int groups, per;
    split_heads(tiles * r.batch, 2 * r.n_kv_heads + r.q.heads, ROPE_WARPS / (D / 128), groups, per);
    const int64_t grid = tiles * r.batch * groups;
    if (grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    const size_t sm = angle_bytes(r.rope);
    const unsigned gr = (unsigned)grid;
    switch (r.kd.type) {
        case 2: rotary_append_kernel<D, T, 2><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per); break;
        case 3: rotary_append_kernel<D, T, 3><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per); break;
        case 4: rotary_append_kernel<D, T, 4><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per); break;
        default: rotary_append_kernel<D, T, 8><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per); break;
    }
    return cudaGetLastError();
}

cudaError_t launch_rotary_append(const RotaryAppendRun& r, cudaStream_t st) {
    if (r.head_dim == 128) {
        if (r.dtype == DT_F32) return launch_append<128, float>(r, st);
        if (r.dtype == DT_F16) return launch_append<128, __half>(r, st);
        return launch_append<128, __nv_bfloat16>(r, st);
    }
    if (r.dtype == DT_F32) return launch_append<256, float>(r, st);
    if (r.dtype == DT_F16) return launch_append<256, __half>(r, st);
    return launch_append<256, __nv_bfloat16>(r, st);
}

cudaError_t launch_dequantize_q8(const int8_t* code, const float* scale, void* y, int out_dtype, int64_t n_blocks,
                                 int head_dim, cudaStream_t st) {
    const int l2 = __builtin_ctz((unsigned)head_dim);   // a block is 16 head_dim codes: head_dim loads
    const int64_t n16 = n_blocks << l2;
    int64_t grid = (n16 + 255) / 256;
    const int64_t most = (int64_t)sm_count() * 32;
    if (grid > most) grid = most;
    const uint4* c = reinterpret_cast<const uint4*>(code);
    if (out_dtype == DT_F32) dequantize_q8_kernel<float><<<(unsigned)grid, 256, 0, st>>>(c, scale, (float*)y, n16, l2);
    else if (out_dtype == DT_F16) dequantize_q8_kernel<__half><<<(unsigned)grid, 256, 0, st>>>(c, scale, (__half*)y, n16, l2);
    else dequantize_q8_kernel<__nv_bfloat16><<<(unsigned)grid, 256, 0, st>>>(c, scale, (__nv_bfloat16*)y, n16, l2);
    return cudaGetLastError();
}

}  // namespace tq
