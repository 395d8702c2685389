// tq_move.cu — rows of a paged cache moved between token slots: the accepted path of a drafted tree, the tokens that an
// eviction keeps.
//
// Row j of (sequence b, KV head h) goes from slot src[b][h][j] to slot first[b] + j: keys and values with their scales,
// and the sums of attention weights.  TurboQuant rows are copied.  An 8-bit block of 16 slots has one scale for rows that
// come from up to 16 blocks: where all of them have the same, codes and scale stay as they are; else
//   scale = max over the rows of max |code| * scale / 127,  code = round(code * old scale / scale),
// the rule by which the append makes them.  Rows of the first block in front of `first` take part in place.
//
// A CTA makes 64 slots (4 blocks of K and of V, a warp each), all in registers: rows are read once and written once.
// What bounds it: instructions of the rescaling, about 6 a code, then the scattered reads.  16 x 8 heads of 8192 kept tokens of 128
// elements in 8 bits with their weights (0.55 GB read and written): 143 us, floor 84 (6 of the 16 sequences: 63 us, issue 67 %, integer
// pipe 60 %, DRAM 32 %); 206 us with conversions by instruction, 166 and 158 us with five and six CTAs an SM, 145 with eight (seven
// spill 8 bytes a thread, eight more).  To other pages, without waits: 118 us of 140 (no weights).  TQ3 rows of 128 elements, the same
// tokens: 123 us; 20 heads of up to 3001 tokens of 256 elements: 16 us with the reading back of the pages.
//
// In place, a slot may be written only after the row that it held has been read.  Slots only fall (src >= first + j,
// checked), so that row is one of the same 64 or of an earlier 64.  CTAs take their 64 in the order in which they start (a
// ticket), read, publish that they have read, and wait for the earlier ones of their (sequence, head) before they write:
// what is waited for has started before and only reads, so every wait ends.  (Two kernels, out to work memory and back, would
// move the bytes twice.)  A wait that runs out all the same ends with TQ_ERROR_TIMEOUT, its rows not written.
#include "leankv_tq.h"
#include "tq_common.cuh"
#include "tq_evict.h"
#include "tq_wait.h"

namespace tq {

constexpr int MOVE_WARPS = 8, MOVE_BLOCKS = 4, MOVE_SLOTS = 16 * MOVE_BLOCKS;

__device__ __forceinline__ uint32_t flag_read(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void flag_write(uint32_t* p, uint32_t v) {
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ uint64_t move_now() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// One warp: until all chunks before `chunk` have been read.  A chunk's flag is 1 when it has been read, 2 when all before
// it have been, too: the way back ends at a 2.
__device__ __forceinline__ bool wait_earlier(const uint32_t* flags, int64_t chunk) {
    const int lane = threadIdx.x & 31;
    for (int64_t base = chunk - 1; base >= 0; base -= 32) {
        const uint64_t until = move_now() + WAIT_NS;
        for (;;) {
            const uint32_t f = base - lane >= 0 ? flag_read(flags + base - lane) : 2u;
            const uint32_t read = __ballot_sync(0xffffffffu, f >= 1), all = __ballot_sync(0xffffffffu, f == 2);
            const int stop = all ? __ffs(all) - 1 : 31;               // the nearest chunk that speaks for the rest
            const uint32_t need = stop == 31 ? 0xffffffffu : (2u << stop) - 1;
            if ((read & need) == need) {
                if (all) return true;
                break;
            }
            if (__any_sync(0xffffffffu, move_now() > until)) return false;
        }
    }
    return true;
}

// where a slot's row lies, as a row of the pool (a row of K and V takes 112 bytes and more, so that 32 bits number all that a GPU
// holds), or NO_ROW: outside the table or the pool
constexpr uint32_t NO_ROW = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t row_at(const MoveRun& r, const int32_t* table, uint32_t cap, int h, uint32_t slot) {
    if (slot >= cap) return NO_ROW;
    const int32_t pg = table[slot >> r.page_shift];
    if (pg < 0 || pg >= r.num_pages) return NO_ROW;
    return (((uint32_t)pg * r.Hkv + h) << r.page_shift) + (slot & ((1u << r.page_shift) - 1));
}

// CTA-wide turn between reading and writing; `used` depends on all that the thread has read, so that the reads are over.
// False: the rows must not be written.
__device__ __forceinline__ bool move_turn(uint32_t* flags, int64_t chunk, uint32_t used, int* s_ok) {
    __syncthreads_or(used == 0x9E3779B9u);
    if (!flags) return true;   // one chunk, or other pages than those that are read
    if (threadIdx.x < 32) {
        if (threadIdx.x == 0) flag_write(flags + chunk, 1u);
        const bool ok = wait_earlier(flags, chunk);
        if (threadIdx.x == 0) {
            if (ok) flag_write(flags + chunk, 2u);
            *s_ok = ok;
        }
    }
    __syncthreads();
    return *s_ok != 0;
}

// What a lane knows of its row (lane & 15) of the warp's block
struct MoveRow {
    uint32_t from = NO_ROW;   // pool row that is read
    bool moved = false;       // one of src (else an older row of the first block, or none)
};

// src, from: of the (sequence, head), the sequence; slots below 2^31, so that differences of them are signed words
__device__ __forceinline__ MoveRow move_row(const MoveRun& r, const int32_t* src, const int32_t* from, uint32_t cap, int h, uint32_t slot, uint32_t to,
                                            uint32_t first, int count, bool q8, bool counts) {
    MoveRow m;
    const int j = (int)(slot - first);
    if (j >= count) return m;
    if (j < 0) {
        if (q8) m.from = to;
        return m;
    }
    const int s = src[j];
    if (s < 0) return m;
    if (to != NO_ROW && !(r.in_place && (uint32_t)s < slot)) m.from = row_at(r, from, cap, h, (uint32_t)s);
    m.moved = m.from != NO_ROW;
    if (!m.moved && counts && r.overflow) atomicAdd(r.overflow, 1);
    return m;
}

// the larger and the smaller of two pairs of 16-bit whole numbers
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.s16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.s16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// round(code * q) of four codes, |code * q| < 127.5: codes as floats from the bits of 2^23 + 128 + code, the product rounded as
// any, then to a whole number by adding 1.5 * 2^23, whose low byte it is (conversions by instruction would go through a unit that
// takes 16 a cycle: 205 us for 16 x 8 heads of 8192 tokens kept)
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, float q) {
    const uint32_t u = codes ^ 0x80808080u;
    const float2 bias = make_float2(-8388736.0f, -8388736.0f), whole = make_float2(12582912.0f, 12582912.0f);
    float2 a = make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7541)));
    float2 b = make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7542)), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7543)));
    a = __fadd2_rn(a, bias);
    b = __fadd2_rn(b, bias);
    // (products one at a time: packed ones are joined with the sums into one rounding)
    a = __fadd2_rn(make_float2(__fmul_rn(a.x, q), __fmul_rn(a.y, q)), whole);
    b = __fadd2_rn(make_float2(__fmul_rn(b.x, q), __fmul_rn(b.y, q)), whole);
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                       __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}

// 8-bit rows of a block: D / 16 lanes a row, 16 codes each
template <int D>
__device__ __forceinline__ void move_block_q8(const MoveRun& r, const MoveSide& x, MoveRow m, uint32_t to0, bool some, uint32_t used,
                                              uint32_t* flags, int64_t chunk, int* s_ok) {
    constexpr int LPR = D / 16, RPP = 32 / LPR, PASSES = 16 / RPP;
    const int lane = threadIdx.x & 31, sub = lane / LPR, col = lane % LPR;
    const bool valid = some && m.from != NO_ROW;
    const uint32_t rows = __ballot_sync(0xffffffffu, valid) & 0xFFFFu;
    const int8_t* pool = reinterpret_cast<const int8_t*>(x.pool);
    uint4 w[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int row = p * RPP + sub;
        const uint32_t from = __shfl_sync(0xffffffffu, m.from, row);
        w[p] = make_uint4(0, 0, 0, 0);
        if ((rows >> row) & 1) w[p] = *reinterpret_cast<const uint4*>(pool + (size_t)from * D + 16 * col);
    }
    const float scale = valid ? x.scale[m.from >> 4] : 0.0f;
    used ^= __float_as_uint(scale);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) used ^= w[p].x ^ w[p].y ^ w[p].z ^ w[p].w;

    // rows' scales alike: nothing changes but the place
    const float one = __shfl_sync(0xffffffffu, scale, rows ? __ffs(rows) - 1 : 0);
    const bool alike = __all_sync(0xffffffffu, !valid || scale == one);
    float now = one;
    if (!alike) {
        float top = 0.0f;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            // largest and least of 16-bit halves whose high bytes are codes (the low ones break ties between equal codes)
            uint32_t most = 0x80008000u, least = 0x7FFF7FFFu;
            const uint32_t in[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                most = max2(most, max2(in[i], in[i] << 8));
                least = min2(least, min2(in[i], in[i] << 8));
            }
            const int hi = max((int)(int16_t)most, (int)most >> 16) >> 8, lo = min((int)(int16_t)least, (int)least >> 16) >> 8;
            const float s = __shfl_sync(0xffffffffu, scale, p * RPP + sub);
            top = fmaxf(top, __fmul_rn(__fmul_rn((float)max(hi, -lo), s), 1.0f / 127.0f));
        }
#pragma unroll
        for (int o = 1; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        now = top >= 0x1p-100f ? top : 0.0f;
    }
    const float ratio = now > 0.0f ? __fdiv_rn(scale, now) : 0.0f;   // of the lane's row
    if (!move_turn(flags, chunk, used, s_ok) || !some) return;
    int8_t* to = reinterpret_cast<int8_t*>(x.pool) + (size_t)to0 * D + 16 * col;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int row = p * RPP + sub;
        const float q = __shfl_sync(0xffffffffu, ratio, row);
        if (!alike) {
            w[p] = make_uint4(rescaled(w[p].x, q), rescaled(w[p].y, q), rescaled(w[p].z, q), rescaled(w[p].w, q));
        }
        if ((rows >> row) & 1) *reinterpret_cast<uint4*>(to + row * D) = w[p];
    }
    if (lane == 0) x.scale[to0 >> 4] = now;
}

// TurboQuant rows of a block: 8 U bytes a row, the block's 16 rows flat over the lanes.  Reading and writing are apart, so that
// the warps of K and of V, whose rows differ in size, meet at one and the same turn between them.
template <int U> constexpr int tq_words() { return (16 * U + 31) / 32; }   // of a lane
template <int U, int M>
__device__ __forceinline__ uint32_t read_block_tq(const MoveSide& x, uint32_t from_row, uint32_t rows, uint2 (&w)[M]) {
    const int lane = threadIdx.x & 31;
    uint32_t used = 0;
#pragma unroll
    for (int i = 0; i < tq_words<U>(); ++i) {
        const int u = lane + 32 * i, row = u < 16 * U ? u / U : 0;
        const uint32_t from = __shfl_sync(0xffffffffu, from_row, row);
        w[i] = make_uint2(0, 0);
        if (u < 16 * U && ((rows >> row) & 1)) w[i] = reinterpret_cast<const uint2*>(x.pool)[(size_t)from * U + u % U];
        used ^= w[i].x ^ w[i].y;
    }
    return used;
}
template <int U, int M>
__device__ __forceinline__ void write_block_tq(const MoveSide& x, uint32_t to0, uint32_t rows, const uint2 (&w)[M]) {
    uint2* to = reinterpret_cast<uint2*>(x.pool) + (size_t)to0 * U;
#pragma unroll
    for (int i = 0; i < tq_words<U>(); ++i) {
        const int u = (threadIdx.x & 31) + 32 * i;
        if (u < 16 * U && ((rows >> (u / U)) & 1)) to[u] = w[i];
    }
}

// D: 8-bit rows of D elements (UK = UV = 0), or TurboQuant rows of 8 UK and 8 UV bytes
template <int D, int UK, int UV>
__global__ void __launch_bounds__(32 * MOVE_WARPS, D == 128 && UK == 0 ? 7 : 4) move_kernel(const MoveRun r, uint32_t chunks) {
    __shared__ uint32_t s_ticket;
    __shared__ int s_ok;
    uint32_t ticket = blockIdx.x;
    if (r.flags) {
        if (threadIdx.x == 0) s_ticket = atomicAdd(r.flags, 1u);
        __syncthreads();
        ticket = s_ticket;
    }
    const uint32_t pairs = (uint32_t)r.B * r.Hkv, chunk = ticket / pairs, pair = ticket - chunk * pairs;
    uint32_t* flags = r.flags ? r.flags + 1 + (size_t)pair * chunks : nullptr;
    const int b = (int)(pair / r.Hkv), h = (int)(pair - (uint32_t)b * r.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, side = warp & 1;
    const uint32_t cap = (uint32_t)(r.max_to << r.page_shift), from_cap = (uint32_t)(r.max_from << r.page_shift);   // at most 2^30
    int first32 = r.first ? r.first[b] : 0, count = (int)r.n;
    if (r.count) count = r.count[b] < 0 ? 0 : (r.count[b] > count ? count : r.count[b]);
    const uint32_t first = first32 < 0 ? 0 : ((uint32_t)first32 > cap ? cap : (uint32_t)first32);

    const uint32_t slot0 = (first & ~15u) + chunk * MOVE_SLOTS + (warp >> 1) * 16;
    const int32_t* to_table = r.to + (int64_t)b * r.max_to;
    const uint32_t to0 = row_at(r, to_table, cap, h, slot0);
    const int row = lane & 15;
    MoveRow m = move_row(r, r.src + ((int64_t)b * r.src_heads + (r.src_heads > 1 ? h : 0)) * r.n, r.from + (int64_t)b * r.max_from, from_cap, h,
                         slot0 + row, to0 == NO_ROW ? NO_ROW : to0 + row, first, count, UK == 0, side == 0 && lane < 16);
    // blocks of rows that all stay where they are, or of none, are left alone
    const bool some = to0 != NO_ROW && __any_sync(0xffffffffu, m.moved && m.from != to0 + row);
    float weight = 0.0f;
    const bool weighs = r.weights && side == 0 && lane < 16 && some && m.moved;
    if (weighs) weight = r.weights[m.from];
    const uint32_t used = __float_as_uint(weight);
    if constexpr (UK == 0) {
        move_block_q8<D>(r, side ? r.v : r.k, m, to0, some, used, flags, chunk, &s_ok);
    } else {
        uint2 w[tq_words<(UK > UV ? UK : UV)>()];
        const uint32_t rows = __ballot_sync(0xffffffffu, some && m.moved) & 0xFFFFu;
        const uint32_t read = side ? read_block_tq<UV>(r.v, m.from, rows, w) : read_block_tq<UK>(r.k, m.from, rows, w);
        const bool go = move_turn(flags, chunk, used ^ read, &s_ok);
        if (go && some) {
            if (side) write_block_tq<UV>(r.v, to0, rows, w);
            else write_block_tq<UK>(r.k, to0, rows, w);
        }
    }
    if (flags && !s_ok) {
        if (threadIdx.x == 0 && r.status) atomicMax(r.status, (int)TQ_ERROR_TIMEOUT);
        return;
    }
    if (weighs) r.weights[to0 + row] = weight;
}

int64_t move_chunks(int64_t n, bool with_first) { return (n + (with_first ? 15 : 0) + MOVE_SLOTS - 1) / MOVE_SLOTS; }

cudaError_t launch_move(const MoveRun& r, cudaStream_t st) {
    const int64_t chunks = move_chunks(r.n, r.first != nullptr), grid = (int64_t)r.B * r.Hkv * chunks;
    if (grid >= (int64_t(1) << 31)) return cudaErrorInvalidConfiguration;
    if (r.flags) {
        const cudaError_t e = cudaMemsetAsync(r.flags, 0, (size_t)(grid + 1) * sizeof(uint32_t), st);
        if (e != cudaSuccess) return e;
    }
    const auto run = [&](auto kernel) {
        kernel<<<(unsigned)grid, 32 * MOVE_WARPS, 0, st>>>(r, (uint32_t)chunks);
        return cudaGetLastError();
    };
    if (r.k.type == 8) return r.D == 256 ? run(move_kernel<256, 0, 0>) : run(move_kernel<128, 0, 0>);
    if (r.D == 256) return r.k.type == 4 ? run(move_kernel<256, 18, 18>) : r.k.type == 3 ? run(move_kernel<256, 14, 18>) : run(move_kernel<256, 10, 18>);
    return r.k.type == 4 ? run(move_kernel<128, 9, 9>) : r.k.type == 3 ? run(move_kernel<128, 7, 9>) : run(move_kernel<128, 5, 9>);
}

}  // namespace tq
