// tq_capi_q8.cu — extern "C" entry points of the rotary operators and the 8-bit paged cache.
#include <cmath>

#include "leankv_tq.h"
#include "tq_attn_q8.h"
#include "tq_capi_internal.h"
#include "tq_common.cuh"
#include "tq_rope.h"

using namespace tq;

// heads of all tensors of a call: their sums and the work split's stay within 32 bits
constexpr int64_t MOST_HEADS = int64_t(1) << 24;

// rows of 8 elements at a time: base and strides on 16-byte boundaries
static tq_status rows_check(const tq_head_rows* x, bool has_dst, size_t eb, const char* name) {
    if (x->heads <= 0) return set_error(TQ_ERROR_INVALID_VALUE, "%s: bad head count", name);
    if (!x->src || (has_dst && !x->dst)) return set_error(TQ_ERROR_INVALID_VALUE, "%s: null pointer", name);
    uintptr_t m = (uintptr_t)x->src | (has_dst ? (uintptr_t)x->dst : 0);
    for (int i = 0; i < 3; ++i)
        m |= (uintptr_t)(x->src_stride[i] * (int64_t)eb) | (has_dst ? (uintptr_t)(x->dst_stride[i] * (int64_t)eb) : 0);
    if (m & 15) return set_error(TQ_ERROR_MISALIGNED, "%s: rows must start on 16-byte boundaries", name);
    if (has_dst && x->src == x->dst)
        for (int i = 0; i < 3; ++i)
            if (x->src_stride[i] != x->dst_stride[i])
                return set_error(TQ_ERROR_INVALID_VALUE, "%s: in place needs equal strides", name);
    return TQ_SUCCESS;
}

static HeadRows rows_of(const tq_head_rows* x) {
    HeadRows r;
    r.src = x->src;
    r.dst = x->dst;
    r.heads = x->heads;
    for (int i = 0; i < 3; ++i) {
        r.ss[i] = x->src_stride[i];
        r.ds[i] = x->dst_stride[i];
    }
    return r;
}

static tq_status rope_check(const tq_rope* p, int head_dim, bool need_positions, Rope* r) {
    if (p->rotary_dim <= 0 || p->rotary_dim > head_dim || p->rotary_dim % 16)
        return set_error(TQ_ERROR_INVALID_VALUE, "rotary_dim=%d (a multiple of 16, at most head_dim)", p->rotary_dim);
    if (!p->inv_freq || (need_positions && !p->positions)) return set_error(TQ_ERROR_INVALID_VALUE, "null frequencies or positions");
    if (p->n_axes <= 0 || p->n_axes > 16) return set_error(TQ_ERROR_INVALID_VALUE, "n_axes=%d (1 .. 16)", p->n_axes);
    if (!std::isfinite(p->scale)) return set_error(TQ_ERROR_INVALID_VALUE, "scale is not finite");
    if (((uintptr_t)p->inv_freq & 7) || (((uintptr_t)p->axis | (uintptr_t)p->positions) & 3))
        return set_error(TQ_ERROR_MISALIGNED, "frequencies, axes or positions not aligned to their element size");
    r->inv_freq = p->inv_freq;
    r->axis = p->axis;
    r->positions = p->positions;
    r->n_axes = p->n_axes;
    r->rotary_dim = p->rotary_dim;
    r->interleaved = p->interleaved != 0;
    r->inverse = p->inverse != 0;
    r->scale = p->scale != 0.0 ? p->scale : 1.0;
    return TQ_SUCCESS;
}

extern "C" tq_status tq_rotary_cuda(const tq_rope* rope, tq_dtype dtype, int batch, int64_t n_new, int head_dim,
                                    const tq_head_rows* x, const tq_head_rows* x2, void* stream) {
    clear_error();
    if (!rope || !x) return set_error(TQ_ERROR_INVALID_VALUE, "null argument");
    if (!dtype_ok(dtype)) return set_error(TQ_ERROR_INVALID_VALUE, "unknown dtype %d", (int)dtype);
    if (batch < 0 || n_new < 0 || n_new > INT32_MAX) return set_error(TQ_ERROR_INVALID_VALUE, "bad batch or token count");
    if (head_dim <= 0 || head_dim % 8 || head_dim > 512)
        return set_error(TQ_ERROR_UNSUPPORTED, "head_dim=%d (a multiple of 8, at most 512)", head_dim);
    RotaryRun r;
    tq_status s = rope_check(rope, head_dim, batch > 0 && n_new > 0, &r.rope);
    if (s) return s;
    if (batch == 0 || n_new == 0) return TQ_SUCCESS;
    if ((int64_t)x->heads + (x2 ? x2->heads : 0) > MOST_HEADS) return set_error(TQ_ERROR_UNSUPPORTED, "more than 2^24 heads");
    if ((s = rows_check(x, true, dtype_bytes(dtype), "x"))) return s;
    if (x2 && (s = rows_check(x2, true, dtype_bytes(dtype), "x2"))) return s;
    r.batch = batch;
    r.head_dim = head_dim;
    r.dtype = (int)dtype;
    r.n_new = n_new;
    r.x[0] = rows_of(x);
    if (x2) r.x[1] = rows_of(x2);
    return cuda_status(launch_rotary(r, (cudaStream_t)stream), "rotary kernel launch");
}

extern "C" tq_status tq_kv_append_rotary_paged_cuda(const tq_rotary_append_args* a, const tq_kv_pages* pg, void* stream) {
    clear_error();
    if (!a) return set_error(TQ_ERROR_INVALID_VALUE, "null argument block");
    if (!dtype_ok(a->dtype)) return set_error(TQ_ERROR_INVALID_VALUE, "unknown dtype %d", (int)a->dtype);
    if (a->batch < 0 || a->n_kv_heads <= 0 || a->n_new < 0 || a->n_new > INT32_MAX)
        return set_error(TQ_ERROR_INVALID_VALUE, "bad batch / head / row counts");
    if (a->head_dim != 128 && a->head_dim != 256)
        return set_error(TQ_ERROR_UNSUPPORTED, "head_dim %d (supported: 128, 256)", a->head_dim);
    const bool q8 = a->k_type == TQ_TYPE_Q8;
    if (q8 ? a->v_type != TQ_TYPE_Q8
           : (a->v_type != TQ_TYPE_TQ4_0 || (a->k_type != TQ_TYPE_TQ4_0 && a->k_type != TQ_TYPE_TQ3_0 && a->k_type != TQ_TYPE_TQ2_0)))
        return set_error(TQ_ERROR_UNSUPPORTED, "block types K=%d V=%d (supported: K TQ4_0, TQ3_0 or TQ2_0 with V TQ4_0, or Q8 for both)",
                         (int)a->k_type, (int)a->v_type);
    int shift = 0;
    tq_status s = pages_check(pg, a->batch, &shift);
    if (s) return s;
    RotaryAppendRun r;
    if (a->rope.inv_freq) {
        if ((s = rope_check(&a->rope, a->head_dim, false, &r.rope))) return s;
        if (a->rope.inverse) return set_error(TQ_ERROR_INVALID_VALUE, "the append rotates forward only");
        if (!a->rope.positions && a->rope.n_axes != 1)
            return set_error(TQ_ERROR_INVALID_VALUE, "several axes need positions");
    } else if (a->q.heads > 0) {
        return set_error(TQ_ERROR_INVALID_VALUE, "queries without a rotation");
    }
    if (a->batch == 0 || a->n_new == 0) return TQ_SUCCESS;
    const size_t eb = dtype_bytes(a->dtype);
    if (a->k.heads != a->n_kv_heads || a->v.heads != a->n_kv_heads)
        return set_error(TQ_ERROR_INVALID_VALUE, "k and v must have n_kv_heads heads");
    if (a->q.heads < 0) return set_error(TQ_ERROR_INVALID_VALUE, "bad query head count");
    if (2 * (int64_t)a->n_kv_heads + a->q.heads > MOST_HEADS) return set_error(TQ_ERROR_UNSUPPORTED, "more than 2^24 heads");
    if ((s = rows_check(&a->k, false, eb, "k")) || (s = rows_check(&a->v, false, eb, "v"))) return s;
    if (a->q.heads > 0 && (s = rows_check(&a->q, true, eb, "q"))) return s;
    if (!a->k_pool || !a->v_pool || (q8 && (!a->k_scale || !a->v_scale))) return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    if (((uintptr_t)a->k_pool | (uintptr_t)a->v_pool) & 15) return set_error(TQ_ERROR_MISALIGNED, "pools must be 16-byte aligned");
    if (((uintptr_t)a->k_scale | (uintptr_t)a->v_scale | (uintptr_t)a->pos | (uintptr_t)a->new_len | (uintptr_t)a->overflow) & 3)
        return set_error(TQ_ERROR_MISALIGNED, "scales, lengths or overflow not 4-byte aligned");
    r.batch = a->batch;
    r.head_dim = a->head_dim;
    r.n_kv_heads = a->n_kv_heads;
    r.dtype = (int)a->dtype;
    r.n_new = a->n_new;
    r.k = rows_of(&a->k);
    r.v = rows_of(&a->v);
    if (a->q.heads > 0) r.q = rows_of(&a->q);
    r.kd.pool = static_cast<uint8_t*>(a->k_pool);
    r.kd.scale = a->k_scale;
    r.kd.type = (int)a->k_type;
    r.vd.pool = static_cast<uint8_t*>(a->v_pool);
    r.vd.scale = a->v_scale;
    r.vd.type = (int)a->v_type;
    r.pages = pg->page_table;
    r.max_pages = pg->max_pages_per_seq;
    r.num_pages = pg->num_pages;
    r.page_shift = shift;
    r.pos = a->pos;
    r.new_len = a->new_len;
    r.rotate = a->rotate != 0;
    r.norm = fwht_norm(a->head_dim);
    r.overflow = a->overflow;
    return cuda_status(launch_rotary_append(r, (cudaStream_t)stream), "rotary append kernel launch");
}

extern "C" tq_status tq_dequantize_q8_cuda(const int8_t* codes, const float* scale, void* y, tq_dtype y_dtype,
                                           int64_t n_blocks, int head_dim, void* stream) {
    clear_error();
    if (!dtype_ok(y_dtype)) return set_error(TQ_ERROR_INVALID_VALUE, "unknown output dtype %d", (int)y_dtype);
    if (head_dim != 128 && head_dim != 256) return set_error(TQ_ERROR_UNSUPPORTED, "head_dim %d (supported: 128, 256)", head_dim);
    if (n_blocks < 0) return set_error(TQ_ERROR_INVALID_VALUE, "n_blocks=%lld", (long long)n_blocks);
    if (n_blocks > (int64_t(1) << 40)) return set_error(TQ_ERROR_UNSUPPORTED, "n_blocks=%lld (at most 2^40)", (long long)n_blocks);
    if (n_blocks == 0) return TQ_SUCCESS;
    if (!codes || !scale || !y) return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    if ((((uintptr_t)codes | (uintptr_t)y) & 15) || ((uintptr_t)scale & 3))
        return set_error(TQ_ERROR_MISALIGNED, "codes and y must be 16-byte aligned, scales 4-byte aligned");
    return cuda_status(launch_dequantize_q8(codes, scale, y, (int)y_dtype, n_blocks, head_dim, (cudaStream_t)stream),
                       "dequantize kernel launch");
}

// ── attention ────────────────────────────────────────────────────────────────

static tq_status q8_check(const tq_attention_q8_args* a, const tq_kv_pages* pg, Q8Run* r, Q8Plan* p) {
    if (!a) return set_error(TQ_ERROR_INVALID_VALUE, "null argument block");
    if (a->batch < 0 || a->n_q_heads <= 0 || a->n_kv_heads <= 0 || a->n_new < 0)
        return set_error(TQ_ERROR_INVALID_VALUE, "bad batch / head / token counts");
    if (a->n_q_heads % a->n_kv_heads) return set_error(TQ_ERROR_INVALID_VALUE, "n_q_heads %% n_kv_heads != 0");
    if (a->head_dim != 128 && a->head_dim != 256)
        return set_error(TQ_ERROR_UNSUPPORTED, "head_dim %d (supported: 128, 256)", a->head_dim);
    if (!dtype_ok(a->q_dtype) || !dtype_ok(a->out_dtype)) return set_error(TQ_ERROR_INVALID_VALUE, "bad dtype");
    int shift = 0;
    tq_status s = pages_check(pg, a->batch, &shift);
    if (s) return s;
    const int64_t cap = pg->max_pages_per_seq << shift, grp = a->n_q_heads / a->n_kv_heads;
    constexpr int64_t MOST = int64_t(1) << 30, MOST_ROWS = int64_t(1) << 40;
    if (pg->max_pages_per_seq > MOST || cap > MOST || a->n_new > MOST || a->n_new * grp > MOST)
        return set_error(TQ_ERROR_UNSUPPORTED, "capacity and rows per head must be at most 2^30");
    // the grid has a CTA for each pair, and the work split's products of rows stay within 64 bits
    const int64_t pairs = (int64_t)a->batch * a->n_kv_heads;
    if (pairs > INT32_MAX || (a->n_new > 0 && pairs > MOST_ROWS / (a->n_new * grp)))
        return set_error(TQ_ERROR_UNSUPPORTED, "batch * n_kv_heads must be below 2^31, query rows at most 2^40");
    if (a->max_kv_len < 0 || a->max_kv_len > cap) return set_error(TQ_ERROR_INVALID_VALUE, "max_kv_len outside [0, capacity]");
    if (!std::isfinite(a->sm_scale)) return set_error(TQ_ERROR_INVALID_VALUE, "sm_scale is not finite");
    r->B = a->batch; r->Hq = a->n_q_heads; r->Hkv = a->n_kv_heads; r->grp = (int)grp; r->D = a->head_dim;
    r->n = a->n_new;
    r->q = a->q; r->q_dtype = (int)a->q_dtype;
    r->out = a->out; r->out_dtype = (int)a->out_dtype;
    for (int i = 0; i < 3; ++i) {
        r->qs[i] = a->q_stride[i];
        r->os[i] = a->out_stride[i];
    }
    r->k = a->k_codes; r->v = a->v_codes; r->ks = a->k_scale; r->vs = a->v_scale;
    r->pages = pg->page_table; r->max_pages = pg->max_pages_per_seq; r->num_pages = pg->num_pages; r->page_shift = shift;
    r->kv_len = a->kv_len; r->q_len = a->q_len;
    r->sm_scale = a->sm_scale != 0.0f ? a->sm_scale : 1.0f / sqrtf((float)a->head_dim);
    r->causal = a->causal != 0; r->rotate_q = a->rotate_q != 0; r->v_rotated = a->v_rotated != 0;
    r->norm = fwht_norm(a->head_dim);
    r->lse = a->lse; r->status = a->status;
    r->max_len = (int)(a->max_kv_len > 0 ? a->max_kv_len : cap);
    *p = q8_plan(a->batch, a->n_kv_heads, (int)grp, a->head_dim, a->n_new, a->max_kv_len > 0 ? a->max_kv_len : cap,
                 a->out_dtype != TQ_DTYPE_BF16);   // a bf16 output has 8 bits: one term of 11 does
    return TQ_SUCCESS;
}

extern "C" size_t tq_attention_q8_workspace_size(const tq_attention_q8_args* a, const tq_kv_pages* pages) {
    clear_error();
    Q8Run r;
    Q8Plan p;
    if (q8_check(a, pages, &r, &p) != TQ_SUCCESS) return 0;
    return q8_workspace_bytes(r.D, p);
}

extern "C" tq_status tq_attention_q8_paged_cuda(const tq_attention_q8_args* a, const tq_kv_pages* pages, void* stream) {
    clear_error();
    Q8Run r;
    Q8Plan p;
    tq_status s = q8_check(a, pages, &r, &p);
    if (s) return s;
    if (r.B == 0 || r.n == 0) return TQ_SUCCESS;
    if (!r.q || !r.out || !r.k || !r.v || !r.ks || !r.vs || !r.kv_len) return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    uintptr_t m = (uintptr_t)r.q | (uintptr_t)r.out | (uintptr_t)r.k | (uintptr_t)r.v;
    for (int i = 0; i < 3; ++i)
        m |= (uintptr_t)(r.qs[i] * (int64_t)dtype_bytes(r.q_dtype)) | (uintptr_t)(r.os[i] * (int64_t)dtype_bytes(r.out_dtype));
    if (m & 15) return set_error(TQ_ERROR_MISALIGNED, "codes and the rows of q and out must start on 16-byte boundaries");
    if (((uintptr_t)r.ks | (uintptr_t)r.vs | (uintptr_t)r.kv_len | (uintptr_t)r.q_len | (uintptr_t)r.lse | (uintptr_t)r.status) & 3)
        return set_error(TQ_ERROR_MISALIGNED, "scales, lengths, lse or status not 4-byte aligned");
    const size_t need = q8_workspace_bytes(r.D, p);
    if (need && (!a->workspace || a->workspace_bytes < need))
        return set_error(TQ_ERROR_INVALID_VALUE, "workspace of %zu bytes needed", need);
    if (need && ((uintptr_t)a->workspace & 15)) return set_error(TQ_ERROR_MISALIGNED, "workspace must be 16-byte aligned");
    if (!r.status && (s = cuda_status(q8_default_status(&r.status), "status word"))) return s;
    return cuda_status(launch_attention_q8(r, p, a->workspace, (cudaStream_t)stream), "attention launch");
}

extern "C" tq_status tq_attention_q8_last_status(int32_t* status, void* stream) {
    clear_error();
    if (!status) return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    *status = 0;
    int32_t* word = nullptr;
    tq_status s = cuda_status(q8_default_status(&word), "status word");
    if (s) return s;
    const cudaStream_t st = (cudaStream_t)stream;
    if ((s = cuda_status(cudaMemcpyAsync(status, word, sizeof *word, cudaMemcpyDeviceToHost, st), "status copy"))) return s;
    if ((s = cuda_status(cudaStreamSynchronize(st), "status copy"))) return s;
    return *status ? cuda_status(cudaMemsetAsync(word, 0, sizeof *word, st), "status clear") : TQ_SUCCESS;
}
