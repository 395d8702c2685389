// tq_capi_evict.cu — extern "C" entry points of drafted trees, sums of attention weights, selection and moving of cached tokens.
#include <cmath>

#include "leankv_tq.h"
#include "tq_capi_internal.h"
#include "tq_common.cuh"
#include "tq_evict.h"

using namespace tq;

constexpr int64_t MOST_TOKENS = int64_t(1) << 30, MOST_PAIRS = INT32_MAX;

extern "C" tq_status tq_draft_tree_cuda(const int32_t* parents, int64_t parents_stride, int batch, int n, uint32_t* mask, int32_t* depth,
                                        void* stream) {
    clear_error();
    if (batch < 0 || n < 0) return set_error(TQ_ERROR_INVALID_VALUE, "bad batch or node count");
    if (batch > 65535 || n > TQ_DRAFT_NODES)
        return set_error(TQ_ERROR_UNSUPPORTED, "%d trees of %d nodes (at most 65535 of %d)", batch, n, TQ_DRAFT_NODES);
    if (batch == 0 || n == 0 || (!mask && !depth)) return TQ_SUCCESS;
    if (!parents) return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    if (((uintptr_t)parents | (uintptr_t)mask | (uintptr_t)depth) & 3) return set_error(TQ_ERROR_MISALIGNED, "parents, masks or depths not 4-byte aligned");
    return cuda_status(launch_draft_tree(parents, parents_stride, batch, n, mask, depth, (cudaStream_t)stream), "tree kernel launch");
}

static bool tq_key_type(int t) { return t == TQ_TYPE_TQ4_0 || t == TQ_TYPE_TQ3_0 || t == TQ_TYPE_TQ2_0; }

// sizes that all calls over pages share; *shift = log2(page_size), *cap = tokens of a sequence
static tq_status sizes_check(int batch, int n_kv_heads, const tq_kv_pages* pg, int* shift, int64_t* cap) {
    if (batch < 0 || n_kv_heads <= 0) return set_error(TQ_ERROR_INVALID_VALUE, "bad batch or head count");
    const tq_status s = pages_check(pg, batch, shift);
    if (s) return s;
    if (pg->max_pages_per_seq > MOST_TOKENS || (pg->max_pages_per_seq << *shift) > MOST_TOKENS)
        return set_error(TQ_ERROR_UNSUPPORTED, "capacity must be at most 2^30 tokens");
    if ((int64_t)batch * n_kv_heads > MOST_PAIRS) return set_error(TQ_ERROR_UNSUPPORTED, "batch * n_kv_heads must be below 2^31");
    *cap = pg->max_pages_per_seq << *shift;
    return TQ_SUCCESS;
}

// ── sums of attention weights ────────────────────────────────────────────────

static tq_status weights_check(const tq_attention_weights_args* a, const tq_kv_pages* pg, WeightsRun* w, WeightsPlan* p) {
    if (!a) return set_error(TQ_ERROR_INVALID_VALUE, "null argument block");
    if (a->n_q_heads <= 0 || a->n_new < 0) return set_error(TQ_ERROR_INVALID_VALUE, "bad head or token counts");
    int shift = 0;
    int64_t cap = 0;
    const tq_status s = sizes_check(a->batch, a->n_kv_heads, pg, &shift, &cap);
    if (s) return s;
    if (a->n_q_heads % a->n_kv_heads) return set_error(TQ_ERROR_INVALID_VALUE, "n_q_heads %% n_kv_heads != 0");
    if (a->head_dim != 128 && a->head_dim != 256)
        return set_error(TQ_ERROR_UNSUPPORTED, "head_dim %d (supported: 128, 256)", a->head_dim);
    if (!dtype_ok(a->q_dtype)) return set_error(TQ_ERROR_INVALID_VALUE, "bad dtype");
    if (a->k_type != TQ_TYPE_Q8 && !tq_key_type(a->k_type)) return set_error(TQ_ERROR_UNSUPPORTED, "keys of type %d", (int)a->k_type);
    const int64_t grp = a->n_q_heads / a->n_kv_heads;
    if (a->n_new > MOST_TOKENS || a->n_new * grp > MOST_TOKENS) return set_error(TQ_ERROR_UNSUPPORTED, "rows per head must be at most 2^30");
    if (a->max_kv_len < 0 || a->max_kv_len > cap) return set_error(TQ_ERROR_INVALID_VALUE, "max_kv_len outside [0, capacity]");
    if (a->window < 0) return set_error(TQ_ERROR_INVALID_VALUE, "window must not be negative");
    if (!std::isfinite(a->sm_scale) || !std::isfinite(a->decay)) return set_error(TQ_ERROR_INVALID_VALUE, "sm_scale or decay is not finite");
    Q8Run& r = w->q;
    r.B = a->batch; r.Hq = a->n_q_heads; r.Hkv = a->n_kv_heads; r.grp = (int)grp; r.D = a->head_dim;
    r.n = a->n_new;
    r.q = a->q; r.q_dtype = (int)a->q_dtype;
    for (int i = 0; i < 3; ++i) r.qs[i] = a->q_stride[i];
    r.k = static_cast<const int8_t*>(a->k_pool); r.ks = a->k_scale;
    r.pages = pg->page_table; r.max_pages = pg->max_pages_per_seq; r.num_pages = pg->num_pages; r.page_shift = shift;
    r.kv_len = a->kv_len; r.q_len = a->q_len;
    r.sm_scale = a->sm_scale != 0.0f ? a->sm_scale : 1.0f / sqrtf((float)a->head_dim);
    r.causal = a->causal != 0; r.rotate_q = a->rotate_q != 0;
    r.norm = fwht_norm(a->head_dim);
    r.status = a->status;
    r.max_len = (int)(a->max_kv_len > 0 ? a->max_kv_len : cap);
    w->k_type = (int)a->k_type;
    w->lse = a->lse;
    w->window = a->window > 0 && a->window < a->n_new ? a->window : a->n_new;
    w->decay = a->decay;
    w->fresh = a->fresh;
    w->weights = a->weights;
    *p = weights_plan(a->batch, a->n_kv_heads, (int)grp, a->head_dim, w->window, r.max_len, a->k_type == TQ_TYPE_Q8);
    return TQ_SUCCESS;
}

extern "C" size_t tq_attention_weights_workspace_size(const tq_attention_weights_args* a, const tq_kv_pages* pages) {
    clear_error();
    WeightsRun w;
    WeightsPlan p;
    return weights_check(a, pages, &w, &p) == TQ_SUCCESS ? p.bytes : 0;
}

extern "C" tq_status tq_attention_weights_paged_cuda(const tq_attention_weights_args* a, const tq_kv_pages* pages, void* stream) {
    clear_error();
    WeightsRun w;
    WeightsPlan p;
    tq_status s = weights_check(a, pages, &w, &p);
    if (s) return s;
    Q8Run& r = w.q;
    if (r.B == 0 || r.max_pages == 0) return TQ_SUCCESS;
    if ((r.n > 0 && (!r.q || !w.lse)) || !r.k || !r.kv_len || !w.weights || (w.k_type == TQ_TYPE_Q8 && !r.ks))
        return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    uintptr_t m = (uintptr_t)r.q | (uintptr_t)r.k | (uintptr_t)w.weights;
    for (int i = 0; i < 3; ++i) m |= (uintptr_t)(r.qs[i] * (int64_t)dtype_bytes(r.q_dtype));
    if (m & 15) return set_error(TQ_ERROR_MISALIGNED, "keys, weights and the rows of q must start on 16-byte boundaries");
    if (((uintptr_t)r.ks | (uintptr_t)r.kv_len | (uintptr_t)r.q_len | (uintptr_t)w.lse | (uintptr_t)w.fresh | (uintptr_t)r.status) & 3)
        return set_error(TQ_ERROR_MISALIGNED, "scales, lengths, lse or status not 4-byte aligned");
    if (p.bytes && (!a->workspace || a->workspace_bytes < p.bytes)) return set_error(TQ_ERROR_INVALID_VALUE, "workspace of %zu bytes needed", p.bytes);
    if (p.bytes && ((uintptr_t)a->workspace & 15)) return set_error(TQ_ERROR_MISALIGNED, "workspace must be 16-byte aligned");
    if (!r.status && (s = cuda_status(q8_default_status(&r.status), "status word"))) return s;
    return cuda_status(launch_weights(w, p, a->workspace, (cudaStream_t)stream), "weights launch");
}

// ── selection ────────────────────────────────────────────────────────────────

extern "C" tq_status tq_select_tokens_cuda(const tq_select_args* a, const tq_kv_pages* pg, void* stream) {
    clear_error();
    if (!a) return set_error(TQ_ERROR_INVALID_VALUE, "null argument block");
    SelectRun r;
    int64_t cap = 0;
    tq_status s = sizes_check(a->batch, a->n_kv_heads, pg, &r.page_shift, &cap);
    if (s) return s;
    if (a->width < 0 || a->sinks < 0 || a->recent < 0) return set_error(TQ_ERROR_INVALID_VALUE, "negative width, sinks or recent");
    if (a->width > MOST_TOKENS) return set_error(TQ_ERROR_UNSUPPORTED, "width must be at most 2^30");
    if (a->max_kv_len < 0 || a->max_kv_len > cap) return set_error(TQ_ERROR_INVALID_VALUE, "max_kv_len outside [0, capacity]");
    if (a->batch == 0 || a->width == 0) return TQ_SUCCESS;
    if (!a->weights || !a->kv_len || !a->slots) return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    if ((uintptr_t)a->weights & 15) return set_error(TQ_ERROR_MISALIGNED, "weights must be 16-byte aligned");
    if (((uintptr_t)a->kv_len | (uintptr_t)a->keep | (uintptr_t)a->slots | (uintptr_t)a->status) & 3)
        return set_error(TQ_ERROR_MISALIGNED, "lengths, slots or status not 4-byte aligned");
    r.B = a->batch; r.Hkv = a->n_kv_heads;
    r.weights = a->weights;
    r.pages = pg->page_table; r.max_pages = pg->max_pages_per_seq; r.num_pages = pg->num_pages;
    r.kv_len = a->kv_len; r.keep = a->keep;
    r.width = a->width; r.sinks = a->sinks; r.recent = a->recent;
    r.max_len = (int)(a->max_kv_len > 0 ? a->max_kv_len : cap);
    r.slots = a->slots;
    r.status = a->status;
    if (!r.status && (s = cuda_status(q8_default_status(&r.status), "status word"))) return s;
    return cuda_status(launch_select(r, (cudaStream_t)stream), "selection launch");
}

// ── moving rows ──────────────────────────────────────────────────────────────

static tq_status move_check(const tq_kv_move_args* a, const tq_kv_pages* pg, MoveRun* r, size_t* bytes) {
    if (!a) return set_error(TQ_ERROR_INVALID_VALUE, "null argument block");
    int64_t cap = 0;
    const tq_status s = sizes_check(a->batch, a->n_kv_heads, pg, &r->page_shift, &cap);
    if (s) return s;
    if (a->head_dim != 128 && a->head_dim != 256)
        return set_error(TQ_ERROR_UNSUPPORTED, "head_dim %d (supported: 128, 256)", a->head_dim);
    if (a->k_type == TQ_TYPE_Q8 ? a->v_type != TQ_TYPE_Q8 : !tq_key_type(a->k_type) || a->v_type != TQ_TYPE_TQ4_0)
        return set_error(TQ_ERROR_UNSUPPORTED, "block types K=%d V=%d (supported: K TQ4_0, TQ3_0 or TQ2_0 with V TQ4_0, or Q8 for both)",
                         (int)a->k_type, (int)a->v_type);
    if (a->n_rows < 0) return set_error(TQ_ERROR_INVALID_VALUE, "n_rows=%lld", (long long)a->n_rows);
    if (a->n_rows > MOST_TOKENS) return set_error(TQ_ERROR_UNSUPPORTED, "n_rows must be at most 2^30");
    if (a->src_heads != 1 && a->src_heads != a->n_kv_heads) return set_error(TQ_ERROR_INVALID_VALUE, "src_heads must be 1 or n_kv_heads");
    if (a->to_table && (a->to_pages_per_seq < 0 || a->to_pages_per_seq > MOST_TOKENS || (a->to_pages_per_seq << r->page_shift) > MOST_TOKENS))
        return set_error(TQ_ERROR_UNSUPPORTED, "capacity must be at most 2^30 tokens");
    r->B = a->batch; r->Hkv = a->n_kv_heads; r->D = a->head_dim;
    r->n = a->n_rows;
    r->src = a->src; r->src_heads = a->src_heads;
    r->first = a->first; r->count = a->count;
    r->k.pool = static_cast<uint8_t*>(a->k_pool); r->k.scale = a->k_scale; r->k.type = (int)a->k_type;
    r->v.pool = static_cast<uint8_t*>(a->v_pool); r->v.scale = a->v_scale; r->v.type = (int)a->v_type;
    r->weights = a->weights;
    r->from = pg->page_table; r->max_from = pg->max_pages_per_seq; r->num_pages = pg->num_pages;
    r->in_place = !a->to_table || a->to_table == pg->page_table;
    r->to = a->to_table ? a->to_table : pg->page_table;
    r->max_to = a->to_table ? a->to_pages_per_seq : pg->max_pages_per_seq;
    r->overflow = a->overflow;
    r->status = a->status;
    if (pg->num_pages >= (int64_t(1) << 32) / (((int64_t)a->n_kv_heads) << r->page_shift))
        return set_error(TQ_ERROR_UNSUPPORTED, "pools must have fewer than 2^32 rows");
    const int64_t chunks = move_chunks(r->n, r->first != nullptr), pairs = (int64_t)r->B * r->Hkv;
    if (pairs > 0 && chunks > INT32_MAX / pairs) return set_error(TQ_ERROR_UNSUPPORTED, "more than 2^37 rows");
    *bytes = r->in_place && chunks > 1 ? (size_t)(pairs * chunks + 1) * sizeof(uint32_t) : 0;
    return TQ_SUCCESS;
}

extern "C" size_t tq_kv_move_workspace_size(const tq_kv_move_args* a, const tq_kv_pages* pages) {
    clear_error();
    MoveRun r;
    size_t bytes = 0;
    return move_check(a, pages, &r, &bytes) == TQ_SUCCESS ? bytes : 0;
}

extern "C" tq_status tq_kv_move_paged_cuda(const tq_kv_move_args* a, const tq_kv_pages* pages, void* stream) {
    clear_error();
    MoveRun r;
    size_t bytes = 0;
    tq_status s = move_check(a, pages, &r, &bytes);
    if (s) return s;
    if (r.B == 0 || r.n == 0) return TQ_SUCCESS;
    const bool q8 = r.k.type == TQ_TYPE_Q8;
    if (!r.src || !r.k.pool || !r.v.pool || (q8 && (!r.k.scale || !r.v.scale))) return set_error(TQ_ERROR_INVALID_VALUE, "null pointer");
    if (((uintptr_t)r.k.pool | (uintptr_t)r.v.pool) & 15) return set_error(TQ_ERROR_MISALIGNED, "pools must be 16-byte aligned");
    if (((uintptr_t)r.k.scale | (uintptr_t)r.v.scale | (uintptr_t)r.src | (uintptr_t)r.first | (uintptr_t)r.count | (uintptr_t)r.weights |
         (uintptr_t)r.to | (uintptr_t)r.overflow | (uintptr_t)r.status) & 3)
        return set_error(TQ_ERROR_MISALIGNED, "scales, slots, lengths, weights, tables, overflow or status not 4-byte aligned");
    if (bytes && (!a->workspace || a->workspace_bytes < bytes)) return set_error(TQ_ERROR_INVALID_VALUE, "workspace of %zu bytes needed", bytes);
    if (bytes && ((uintptr_t)a->workspace & 3)) return set_error(TQ_ERROR_MISALIGNED, "workspace must be 4-byte aligned");
    r.flags = bytes ? static_cast<uint32_t*>(a->workspace) : nullptr;
    if (!r.status && (s = cuda_status(q8_default_status(&r.status), "status word"))) return s;
    return cuda_status(launch_move(r, (cudaStream_t)stream), "move launch");
}
