// tq_rope.cu — rotation of head rows by position, alone and fused into the paged append.
//
// Kernels
//   rotary_kernel<T>                  queries and keys rotated (or rotated back) into strided outputs
//   rotary_append_kernel<D, T, KT>    keys: rotate by position, Hadamard, quantize into pages; values: Hadamard,
//                                     quantize into pages; queries: rotate.  One launch for all three.
//   dequantize_q8_kernel<T>           values of 8-bit pages
//
// Angles.  A pair turns by p * f with p an integer position, so only the fraction of p * f / 2 pi matters.  F =
// floor(f / (2 pi) * 2^64) is within 2^-64 of a turn, and p * F mod 2^64 is that fraction within p 2^-64: 3.4e-13
// radians at a million positions, 7.3e-10 at 2^31, for every f.  (The 64-bit product p * f rounds to 2^-53 of itself:
// 1.2e-10 at a million radians, and less than p 2^-64 turns where f is below 2 pi 2^-11 = 0.003.)  The fraction is
// folded to an eighth of a turn and its sine and cosine are Taylor sums in 64 bits (the next term is below 2^-54),
// rounded once to 32 bits: at a million positions, values near 1 are the true ones' rounding but for one in some 10^5
// that lie that near to a border.  64-bit library functions of the 64-bit product differ where either's error shows:
// of 41537 random calls, 35 had an element of a rotated row one step of its 16-bit type apart, and none a quantized
// code.  They cost about 60 instructions for a pair; a CTA takes 16 tokens and keeps their angles in shared memory for
// all its heads.
//
// Bit-exactness: rotation, Hadamard stages and quantization are single fp32 operations, each correctly
// rounded, in the order of the separate operations (x c - y s with three roundings, stages h = 1, 2, 4, ...).
#include <type_traits>

#include "tq_common.cuh"
#include "tq_kernels.h"
#include "tq_near.cuh"
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

// Rotates `count` rows, `src_step` elements apart, row k by the angles of table row tab_row + k * tab_step: the
// tokens of one head (tab_step 1) or the heads of one token (0).  An item is one row's pair of 8-element runs that
// turn into each other (c and c + R / 16 runs on), or two runs that are only copied.  Every element is read and
// written by one thread, so dst may be src.
template <typename T, int BATCH>
__device__ __forceinline__ void rope_rows(const T* __restrict__ src, int64_t src_step, T* dst, int64_t dst_step, int D,
                                          const Rope& rope, const float2* __restrict__ tab, int count, int tab_row,
                                          int tab_step, int lane, int lanes) {
    const int R = rope.rotary_dim, n8 = ((R >> 1) + 7) >> 3, half8 = R >> 4;
    const int per = (D + 15) >> 4;   // items per row
    const int items = count * per;
    // items of a lane: BATCH at a time, so that their loads are under way together
    for (int first = lane; first < items; first += BATCH * lanes) {
        Raw8<T> a[BATCH], b[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int it = first + i * lanes;
            if (it >= items) break;
            const int k = it / per, c = it % per;
            const T* s = src + k * src_step;
            const T* d = dst + k * dst_step;
            const bool apart = c < half8 && !rope.interleaved;
            if (c >= half8 && s == d) continue;
            const int lo = apart ? 8 * c : 16 * c, hi = apart ? 8 * c + (R >> 1) : 16 * c + 8;
            a[i] = load_raw8<T>(s + lo);
            if (hi < D) b[i] = load_raw8<T>(s + hi);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int it = first + i * lanes;
            if (it >= items) break;
            const int k = it / per, c = it % per, row = tab_row + k * tab_step;
            const T* s = src + k * src_step;
            T* d = dst + k * dst_step;
            if (c >= half8 && s == d) continue;
            const bool apart = c < half8 && !rope.interleaved;
            const int lo = apart ? 8 * c : 16 * c, hi = apart ? 8 * c + (R >> 1) : 16 * c + 8;
            if (c >= half8) {
                store_raw8<T>(d + lo, a[i]);
                if (hi < D) store_raw8<T>(d + hi, b[i]);
                continue;
            }
            float x[8], y[8];
            unpack8(a[i], x);
            unpack8(b[i], y);
            if (apart) {
                float cs[8], sn[8];
                angles8(tab, row, c, n8, cs, sn);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float u = x[j], w = y[j];
                    x[j] = rot_lo(u, w, cs[j], sn[j]);
                    y[j] = rot_hi(u, w, cs[j], sn[j]);
                }
            } else {
                turn_neighbours(x, tab, row, 2 * c, n8);
                turn_neighbours(y, tab, row, 2 * c + 1, n8);
            }
            store8<T>(d + lo, x);
            store8<T>(d + hi, y);
        }
    }
}

// The warp's share of a tile's rows [r0, r1) of `heads` heads: whole heads, or whole tokens where a token's heads
// lie together in memory (a warp then reads a run of heads * D elements).
template <typename T, int BATCH>
__device__ __forceinline__ void rope_heads(const HeadRows& x, int b, int64_t t0, int r0, int r1, int h0, int h1, bool by_token,
                                           int D, const Rope& rope, const float2* __restrict__ tab, int part, int parts) {
    const int lane = threadIdx.x & 31;
    const T* src = static_cast<const T*>(x.src) + b * x.ss[0] + t0 * x.ss[2];
    T* dst = static_cast<T*>(x.dst) + b * x.ds[0] + t0 * x.ds[2];
    if (by_token) {
        for (int row = r0 + part; row < r1; row += parts)
            rope_rows<T, BATCH>(src + row * x.ss[2] + h0 * x.ss[1], x.ss[1], dst + row * x.ds[2] + h0 * x.ds[1], x.ds[1], D, rope, tab,
                                h1 - h0, row, 0, lane, 32);
    } else {
        for (int h = h0 + part; h < h1; h += parts)
            rope_rows<T, BATCH>(src + r0 * x.ss[2] + h * x.ss[1], x.ss[2], dst + r0 * x.ds[2] + h * x.ds[1], x.ds[2], D, rope, tab,
                                r1 - r0, r0, 1, lane, 32);
    }
}
// tokens of one head lie further apart than the heads of one token
__device__ __forceinline__ bool token_major(const HeadRows& x) { return x.ss[1] < x.ss[2] && x.ss[1] > 0; }

// CTAs per SM: 64 registers are enough for bf16 (8192 tokens of 40 heads: 65 us, with 80 registers 73 us); the
// conversions of f16 spill there (4551 tokens of 18 wide heads: 34 us, with 80 registers 25 us)
template <typename T> constexpr int ROTARY_CTAS = std::is_same<T, __nv_bfloat16>::value ? 4 : 3;

template <typename T>
__global__ void __launch_bounds__(ROPE_THREADS, ROTARY_CTAS<T>) rotary_kernel(const RotaryRun r, int tiles, int groups, int per_group) {
    extern __shared__ __align__(16) uint8_t smem[];
    float2* tab = reinterpret_cast<float2*>(smem);
    const int g = blockIdx.x % groups, tile = (blockIdx.x / groups) % tiles, b = blockIdx.x / groups / tiles;
    const int64_t t0 = (int64_t)tile * ROPE_TOKENS;
    const int rows = (int)(r.n_new - t0 < ROPE_TOKENS ? r.n_new - t0 : ROPE_TOKENS);
    fill_angles(tab, r.rope, b, r.batch, t0, r.n_new, 0);
    __syncthreads();
    const int warp = threadIdx.x >> 5;
    // heads [g per_group, ...) of the list x[0] | x[1]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int first = i ? r.x[0].heads : 0;
        int h0 = g * per_group - first, h1 = h0 + per_group;
        h0 = h0 < 0 ? 0 : h0;
        h1 = h1 > r.x[i].heads ? r.x[i].heads : h1;
        if (h0 < h1)
            rope_heads<T, 2>(r.x[i], b, t0, 0, rows, h0, h1, rows >= ROPE_WARPS && token_major(r.x[i]), r.head_dim,
                                                  r.rope, tab, warp, ROPE_WARPS);
    }
}

// ── append ─────────────────────────────────────────────────────────────────

// A lane holds elements 8 i .. 8 i + 7 and D / 2 + 8 i .. of a row (v[0 .. 7], v[8 .. 15]), so that the halves of a
// pair (i, i + D / 2) meet in one lane.  Hadamard stages in the reference's order: h = 1, 2, 4 within 8 elements,
// h = 8 .. D / 4 between lanes, h = D / 2 between the two runs; each a correctly rounded sum and difference, then
// the factor 1 / sqrt(D).
template <int D>
__device__ __forceinline__ void fwht_halves(float (&v)[16], float norm) {
    const float2 m1 = make_float2(-1.0f, -1.0f);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        const float a = v[j], b = v[j + 1];
        v[j] = __fadd_rn(a, b);
        v[j + 1] = __fsub_rn(a, b);
    }
#pragma unroll
    for (int h = 2; h < 8; h *= 2) {
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            if (j & h) continue;
            const float2 a = make_float2(v[j], v[j + 1]), b = make_float2(v[j + h], v[j + h + 1]);
            const float2 s = __fadd2_rn(a, b), d = __ffma2_rn(b, m1, a);
            v[j] = s.x; v[j + 1] = s.y; v[j + h] = d.x; v[j + h + 1] = d.y;
        }
    }
#pragma unroll
    for (int bit = 1; bit < D / 16; bit *= 2) {
        const float sg = (threadIdx.x & bit) ? -1.0f : 1.0f;   // lower: self + other, upper: other - self
        const float2 sg2 = make_float2(sg, sg);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float p0 = __shfl_xor_sync(0xffffffffu, v[j], bit), p1 = __shfl_xor_sync(0xffffffffu, v[j + 1], bit);
            const float2 s = __ffma2_rn(make_float2(v[j], v[j + 1]), sg2, make_float2(p0, p1));
            v[j] = s.x; v[j + 1] = s.y;
        }
    }
    const float2 n2 = make_float2(norm, norm);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float2 a = make_float2(v[j], v[j + 1]), b = make_float2(v[j + 8], v[j + 9]);
        const float2 s = __fmul2_rn(__fadd2_rn(a, b), n2), d = __fmul2_rn(__ffma2_rn(b, m1, a), n2);
        v[j] = s.x; v[j + 1] = s.y; v[j + 8] = d.x; v[j + 9] = d.y;
    }
}

// elements e .. e + 7 of a key row, turned (any rotary_dim and pairing); a partner run is read from the row again
template <typename T>
__device__ __forceinline__ void turned8(const T* __restrict__ row_ptr, int e, const Rope& rope,
                                        const float2* __restrict__ tab, int row, int n8, float* v8) {
    float v[8];
    load8<T>(row_ptr + e, v);
    const int R = rope.rotary_dim;
    if (e < R && rope.interleaved) {
        turn_neighbours(v, tab, row, e >> 3, n8);
    } else if (e < R) {
        const int hi = e >= (R >> 1);
        const int c = (hi ? e - (R >> 1) : e) >> 3;
        float p[8], cs[8], sn[8];
        load8<T>(row_ptr + (hi ? e - (R >> 1) : e + (R >> 1)), p);
        angles8(tab, row, c, n8, cs, sn);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = hi ? rot_hi(p[j], v[j], cs[j], sn[j]) : rot_lo(v[j], p[j], cs[j], sn[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v8[j] = v[j];
}

// Packs this lane's 8 codes (elements 8 a .. 8 a + 7 of a 32-element block, a = lane & 3) into the staged block.
template <int QT>
__device__ __forceinline__ void stage_quarter_block(uint8_t* __restrict__ blk, const uint32_t* code, int a, uint16_t d) {
    if (a == 0) *reinterpret_cast<uint16_t*>(blk) = d;
    if constexpr (QT == 4) {
        // byte j = code j | code j + 16 << 4: lanes a and a + 2 hold the nibbles of bytes 8 a .. 8 a + 7; the lower
        // lane writes the first four of them, the upper lane the others
        uint32_t own = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) own |= code[j] << (4 * j);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 2);
        const uint32_t lo = (a < 2 ? own : other >> 16) & 0xFFFFu, hi = (a < 2 ? other : own >> 16) & 0xFFFFu;
        uint16_t* w = reinterpret_cast<uint16_t*>(blk + 2 + 8 * (a & 1) + 4 * (a >> 1));
        // nibbles n0 .. n3 of each to the low and high halves of four bytes
        const uint32_t l0 = lo & 0xFFu, l1 = lo >> 8, h0 = hi & 0xFFu, h1 = hi >> 8;
        w[0] = (uint16_t)((l0 & 15u) | ((h0 & 15u) << 4) | ((l0 >> 4) << 8) | ((h0 >> 4) << 12));
        w[1] = (uint16_t)((l1 & 15u) | ((h1 & 15u) << 4) | ((l1 >> 4) << 8) | ((h1 >> 4) << 12));
    } else if constexpr (QT == 3) {
        // 24 bits at byte 3 a: an even lane writes its first two bytes and its last with the odd lane's first
        uint32_t g = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) g |= code[j] << (3 * j);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, g, 1);
        uint16_t* w = reinterpret_cast<uint16_t*>(blk + 2 + 6 * (a >> 1));
        if (a & 1) {
            w[2] = (uint16_t)(g >> 8);
        } else {
            w[0] = (uint16_t)g;
            w[1] = (uint16_t)((g >> 16) | ((other & 0xFFu) << 8));
        }
    } else {
        uint32_t g = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) g |= code[j] << (2 * j);
        reinterpret_cast<uint16_t*>(blk + 2)[a] = (uint16_t)g;
    }
}

// codes of 8 elements of a block whose maximum is amax; near: shared address of the level table, or 0 (few rows: the
// comparisons cost less than the table)
template <int QT>
__device__ __forceinline__ void nearest8(const float* v, float amax, uint32_t near, uint32_t* code) {
    const float inv = amax > 0.0f ? __fdiv_rn(1.0f, amax) : 0.0f;
    if (near != 0 && inv != INFINITY) {
#pragma unroll
        for (int j = 0; j < 8; j += 2)
            near_pair(__fmul2_rn(make_float2(v[j], v[j + 1]), make_float2(inv, inv)), near, code[j], code[j + 1]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float xn = __fmul_rn(v[j], inv);
        code[j] = (uint32_t)(QT == 4 ? tq4_nearest(xn) : QT == 3 ? tq3_nearest(xn) : tq2_nearest(xn));
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
                                            float* __restrict__ s_amax, uint32_t near, int sub, int bar) {
    constexpr int LPR = D / 16, RPP = 32 / LPR, WPU = D / 128, RPW = 16 / WPU, PASSES = RPW / RPP;
    const int lane = threadIdx.x & 31, lr = lane / LPR, li = lane % LPR;
    const int64_t at = tile_rows_at(r, b, h, slot0);
    if (at < 0) {
        if (r.overflow && lane == 0 && sub == 0) atomicAdd(r.overflow, rb - ra);
        return;
    }
    const T* src = static_cast<const T*>(x.src) + b * x.ss[0] + h * x.ss[1] + t0 * x.ss[2];
    const int n8 = ((r.rope.rotary_dim >> 1) + 7) >> 3;
    // halves of the whole head turn into each other: the lane has both; else their runs are read where they lie
    const bool halves = !turn || (r.rope.rotary_dim == D && !r.rope.interleaved);
    auto has_rows = [&](int p) {   // the same for all lanes
        const int base = sub * RPW + p * RPP;
        return base + RPP > ra && base < rb;
    };
    auto load = [&](int p, Raw8<T>& lo, Raw8<T>& hi) {
        const int row = sub * RPW + p * RPP + lr;
        if (row >= ra && row < rb) {
            const T* q = src + row * x.ss[2] + 8 * li;
            lo = load_raw8<T>(q);
            hi = load_raw8<T>(q + D / 2);
        }
    };
    auto values = [&](int p, const Raw8<T>& lo, const Raw8<T>& hi, float (&v)[16]) {
        const int row = sub * RPW + p * RPP + lr;
        if (row >= ra && row < rb) {
            if (halves) {
                float a[8], c[8];
                unpack8(lo, a);
                unpack8(hi, c);
                if (turn) {
                    float cs[8], sn[8];
                    angles8(tab, row, li, n8, cs, sn);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[j] = rot_lo(a[j], c[j], cs[j], sn[j]);
                        v[8 + j] = rot_hi(a[j], c[j], cs[j], sn[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) { v[j] = a[j]; v[8 + j] = c[j]; }
                }
            } else {
                turned8<T>(src + row * x.ss[2], 8 * li, r.rope, tab, row, n8, v);
                turned8<T>(src + row * x.ss[2], D / 2 + 8 * li, r.rope, tab, row, n8, v + 8);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.0f;
        }
        if (r.rotate) fwht_halves<D>(v, r.norm);
    };

    if constexpr (QT == 8) {
        float v[PASSES][16];
        float amax = 0.0f;
        {
#pragma unroll
            for (int p = 0; p < PASSES; ++p) {
                Raw8<T> lo, hi;
                if (has_rows(p)) load(p, lo, hi);
                if (!has_rows(p)) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[p][j] = 0.0f;
                    continue;
                }
                values(p, lo, hi, v[p]);
#pragma unroll
                for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(v[p][j]));
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        float* sp = dst.scale + (at >> 4);
        // read by the lane that stores the new scale below, so that no lane can meet the new one
        float s_old = 0.0f;
        if (older > 0 && lane == 0) s_old = *sp;
        s_old = __shfl_sync(0xffffffffu, s_old, 0);
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
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint2* cell = reinterpret_cast<uint2*>(pool + row * D + half * (D / 2) + 8 * li);
                uint32_t w[2];
                if (row >= ra && row < rb) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t acc = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            int c = __float2int_rn(__fmul_rn(v[p][8 * half + 4 * i + j], inv));
                            c = c < -127 ? -127 : (c > 127 ? 127 : c);
                            acc |= (uint32_t)(c & 0xFF) << (8 * j);
                        }
                        w[i] = acc;
                    }
                    *cell = make_uint2(w[0], w[1]);
                } else if (grow && row < older) {
                    const uint2 o = *cell;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t acc = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int c = (int)(int8_t)((i ? o.y : o.x) >> (8 * j));
                            acc |= (uint32_t)(__float2int_rn(__fmul_rn((float)c, ratio)) & 0xFF) << (8 * j);
                        }
                        w[i] = acc;
                    }
                    *cell = make_uint2(w[0], w[1]);
                }
            }
        }
        if (lane == 0 && sub == 0 && (older == 0 || s != s_old)) *sp = s;
    } else {
        constexpr int BB = BlockBytes<QT>::value, ROWB = D / 32 * BB;
        Raw8<T> lo, hi;
        if (has_rows(0)) load(0, lo, hi);
#pragma unroll 1
        for (int p = 0; p < PASSES; ++p) {
            float v[16];
            const bool some = has_rows(p);
            if (some) values(p, lo, hi, v);
            if (p + 1 < PASSES && has_rows(p + 1)) load(p + 1, lo, hi);   // the next rows, under this pass's search
            if (!some) continue;
            const int row = p * RPP + lr;   // staged row
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float amax = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[8 * half + j]));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                uint32_t code[8];
                nearest8<QT>(v + 8 * half, amax, near, code);
                stage_quarter_block<QT>(stage + row * ROWB + (half * (LPR / 4) + (li >> 2)) * BB, code, li & 3, half_trunc(amax));
            }
        }
        __syncwarp();
        // the new rows are consecutive slots of one page: one run of 8-byte words
        const int first = ra > sub * RPW ? ra : sub * RPW, last = rb < (sub + 1) * RPW ? rb : (sub + 1) * RPW;
        const uint2* from = reinterpret_cast<const uint2*>(stage + (first - sub * RPW) * ROWB);
        uint2* to = reinterpret_cast<uint2*>(dst.pool + (at + first) * ROWB);
        for (int i = lane; i < (last - first) * (ROWB / 8); i += 32) to[i] = from[i];
        __syncwarp();
    }
}

// CTAs per SM: 80 registers spill a few bytes of the TQ encoders' for 16-bit rows, and the third CTA hides more of
// their chains (16384 tokens of 8 + 8 and 32 query heads: 100 us, 111 with two CTAs, 107 with four; a token of 64
// sequences 10.4, 11.5 and 11.9 us).  32-bit rows (8192 tokens: 102 us with three, 83 with two) and the 8-bit pages'
// kernels (4 x 2000 tokens: 46.7 and 44.9 us) spill too much.
template <typename T, int KT> constexpr int APPEND_CTAS = KT != 8 && sizeof(T) == 2 ? 3 : 2;

// Work of a CTA: 16 slot-aligned tokens of one sequence, heads [g * per_group, ...) of the list
// K heads | V heads | query heads.  The slot alignment gives an 8-bit scale block to one unit.
template <int D, typename T, int KT>
__global__ void __launch_bounds__(ROPE_THREADS, APPEND_CTAS<T, KT>)
rotary_append_kernel(const RotaryAppendRun r, int tiles, int groups, int per_group, int tables) {
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
    if (turn) fill_angles(tab, r.rope, b, r.batch, t0, r.n_new, pos);
    // level tables of the key and the value type behind the angles
    uint32_t near_k = 0, near_v = 0;
    if (KT != 8 && tables) {
        uint2* t = reinterpret_cast<uint2*>(smem + tables);
        near_table_init<KT == 8 ? 4 : KT, ROPE_THREADS>(t);
        if (KT != 4) near_table_init<4, ROPE_THREADS>(t + NEAR_ROWS * NEAR_REP);
        near_k = (uint32_t)__cvta_generic_to_shared(t) + 8u * (threadIdx.x & (NEAR_REP - 1));
        near_v = near_k + (KT != 4 ? NEAR_ROWS * NEAR_REP * (uint32_t)sizeof(uint2) : 0u);
    }
    __syncthreads();
    const int ra = t0 < 0 ? (int)-t0 : 0;
    const int rb = len - t0 < ROPE_TOKENS ? (int)(len - t0) : ROPE_TOKENS;        // stored rows of the tile
    const int rq = r.n_new - t0 < ROPE_TOKENS ? (int)(r.n_new - t0) : ROPE_TOKENS;   // query rows
    const int warp = threadIdx.x >> 5, sub = warp % WPU;
    // heads [g per_group, ...) of the list K | V | queries
    const int Hkv = r.n_kv_heads, total = 2 * Hkv + r.q.heads;
    const int first = g * per_group, end = first + per_group < total ? first + per_group : total;
    const int slots = ROPE_WARPS / WPU, slot = warp / WPU;
    for (int u = first + slot; u < end && u < 2 * Hkv; u += slots) {
        uint8_t* stage = s_stage + (KT == 8 ? 0 : warp * STAGE_BYTES);
        float* am = s_amax + (warp - sub);
        const int bar = 1 + slot;
        if (ra >= rb) continue;
        if (u < Hkv) append_unit<D, T, KT>(r, r.k, r.kd, turn, b, u, slot0, t0, ra, rb, ra, tab, stage, am, near_k, sub, bar);
        else append_unit<D, T, VT>(r, r.v, r.vd, false, b, u - Hkv, slot0, t0, ra, rb, ra, tab, stage, am, near_v, sub, bar);
    }
    const int h0 = first > 2 * Hkv ? first - 2 * Hkv : 0, h1 = end - 2 * Hkv;
    if (h0 < h1) {
        // the warps that have taken one K or V head fewer begin
        const int taken = first < 2 * Hkv ? (2 * Hkv - first) % slots * WPU : 0;
        const int part = (warp + ROPE_WARPS - taken) % ROPE_WARPS;
        rope_heads<T, sizeof(T) == 2 ? 2 : 1>(r.q, b, t0, ra, rq, h0, h1, rq - ra >= ROPE_WARPS && token_major(r.q), D, r.rope, tab, part,
                                              ROPE_WARPS);
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
// spreads its heads over CTAs instead (down to one unit per warp) until the grid covers the SMs twice.  Where the tiles
// cover them once, a split that leaves the last CTA under half of the others' heads only adds angles and an uneven
// end (285 tiles of 18 heads of 256: 30 us as 16 + 2, 20 us whole; 188 tiles: 23 and 19 us).
static void split_heads(int64_t tiles, int total, int slots, int& groups, int& per_group) {
    const int64_t want = 2 * (int64_t)sm_count();
    int64_t g = (want + tiles - 1) / tiles;
    const int most = (total + slots - 1) / slots;
    if (g > most) g = most;
    if (g < 1) g = 1;
    per_group = (int)((total + g - 1) / g);
    per_group = (per_group + slots - 1) / slots * slots;
    groups = (total + per_group - 1) / per_group;
    if (tiles >= sm_count() && 2 * (total - (groups - 1) * per_group) < per_group) {
        groups = 1;
        per_group = total;
    }
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
    // The level tables (8 KB each) pay when a warp has units of full tiles to search: a 16384-token prompt of 8 + 8
    // heads and 32 query heads took 100 us with them and 115 us without.  Steps of a few tokens take comparisons.
    const size_t angles = (angle_bytes(r.rope) + 127) & ~size_t(127);
    const bool table = r.kd.type != 8 && r.n_new >= ROPE_TOKENS;
    const int at = table ? (int)(angles > 0 ? angles : 128) : 0;
    const size_t sm = table ? at + (size_t)NEAR_ROWS * NEAR_REP * sizeof(uint2) * (r.kd.type == 4 ? 1 : 2) : angles;
    const unsigned gr = (unsigned)grid;
    switch (r.kd.type) {
        case 2: rotary_append_kernel<D, T, 2><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per, at); break;
        case 3: rotary_append_kernel<D, T, 3><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per, at); break;
        case 4: rotary_append_kernel<D, T, 4><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per, at); break;
        default: rotary_append_kernel<D, T, 8><<<gr, ROPE_THREADS, sm, st>>>(r, (int)tiles, groups, per, at); break;
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
