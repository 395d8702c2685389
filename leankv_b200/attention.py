"""Fused attention over packed TurboQuant K/V caches and 8-bit pages (torch front end).

Cache tensors are uint8 with shape [batch, n_kv_heads, capacity, head_dim/32, bytes]
of TQ4_0 (18-byte) or, for K, TQ3_0 (14-byte) or TQ2_0 (10-byte) blocks (src/ggml-tq.h:125-141);
head_dim is 128 or 256 and capacity even.  K and V hold Hadamard-rotated rows
(quantize with fwht_head_dim=head_dim); the query is rotated inside, and the
output rotated back, so the result is attention in the original space.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib as L
from .ops import (_DTYPES, _PAGES, _TYPE_OF_BYTES, DraftTree, _call, _check_lengths, _check_q8_pools, _check_rows, _check_status,
                  _check_table, _check_weights, _device_of, _need_cuda, _own_rows, _row_strides, _stream, _work_bytes)


class AttnArgs(C.Structure):
    """Mirror of tq_decode_attention_args (include/leankv_tq.h)."""
    _fields_ = [
        ("batch", C.c_int), ("n_q_heads", C.c_int), ("n_kv_heads", C.c_int), ("head_dim", C.c_int),
        ("q", C.c_void_p), ("q_dtype", C.c_int),
        ("k_cache", C.c_void_p), ("k_type", C.c_int),
        ("v_cache", C.c_void_p), ("v_type", C.c_int),
        ("kv_capacity", C.c_int64),
        ("kv_len", C.c_void_p),
        ("max_kv_len", C.c_int64),
        ("sm_scale", C.c_float),
        ("rotate_q", C.c_int),
        ("v_rotated", C.c_int),
        ("out", C.c_void_p), ("out_dtype", C.c_int),
        ("lse", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class KVPages(C.Structure):
    """Mirror of tq_kv_pages (include/leankv_tq.h): a paged cache's page table."""
    _fields_ = [("page_table", C.c_void_p), ("max_pages_per_seq", C.c_int64), ("num_pages", C.c_int64),
                ("page_size", C.c_int)]


def make_pages(page_table: torch.Tensor, num_pages: int, page_size: int) -> KVPages:
    pg = KVPages()
    pg.page_table = page_table.data_ptr()
    pg.max_pages_per_seq = page_table.shape[1]
    pg.num_pages = int(num_pages)
    pg.page_size = int(page_size)
    return pg


def _bind():
    lib = L.load()
    lib.tq_decode_attention_workspace_size.restype = C.c_size_t
    lib.tq_decode_attention_workspace_size.argtypes = [C.POINTER(AttnArgs)]
    lib.tq_decode_attention_cuda.restype = C.c_int
    lib.tq_decode_attention_cuda.argtypes = [C.POINTER(AttnArgs), C.c_void_p]
    lib.tq_decode_attention_paged_cuda.restype = C.c_int
    lib.tq_decode_attention_paged_cuda.argtypes = [C.POINTER(AttnArgs), C.POINTER(KVPages), C.c_void_p]
    lib.tq_lse_combine_cuda.restype = C.c_int
    lib.tq_lse_combine_cuda.argtypes = [C.c_int, C.c_int64, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p,
                                        C.c_void_p, C.c_void_p]
    return lib


_workspaces: dict = {}


def _workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    key = (device.type, device.index)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def make_args(q, k_cache, v_cache, kv_len=None, max_kv_len=0, sm_scale=0.0, rotate_q=True, v_rotated=True,
              out=None, lse=None, k_type=4, v_type=4):
    B, Hq, D = q.shape
    Hkv, cap = k_cache.shape[1], k_cache.shape[2]
    a = AttnArgs()
    a.batch, a.n_q_heads, a.n_kv_heads, a.head_dim = B, Hq, Hkv, D
    a.q, a.q_dtype = q.data_ptr(), _DTYPES[q.dtype]
    a.k_cache, a.k_type = k_cache.data_ptr(), k_type
    a.v_cache, a.v_type = v_cache.data_ptr(), v_type
    a.kv_capacity = cap
    a.kv_len = kv_len.data_ptr() if kv_len is not None else None
    a.max_kv_len = int(max_kv_len)
    a.sm_scale = float(sm_scale)
    a.rotate_q, a.v_rotated = int(rotate_q), int(v_rotated)
    a.out, a.out_dtype = out.data_ptr(), _DTYPES[out.dtype]
    a.lse = lse.data_ptr() if lse is not None else None
    return a


def decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     kv_len: torch.Tensor | None = None, max_kv_len: int | None = None,
                     sm_scale: float | None = None, rotate_q: bool = True, v_rotated: bool = True,
                     out_dtype: torch.dtype = torch.float32, return_lse: bool = False,
                     out: torch.Tensor | None = None, lse_out: torch.Tensor | None = None):
    """softmax(q~ K^T * sm_scale) V over packed caches; q [B, Hq, D] -> out [B, Hq, D].

    kv_len: int32 CUDA tensor [B] of valid tokens (default: the whole capacity);
    max_kv_len: host-side upper bound of kv_len used to plan the split-KV work
    (default: the capacity).  out / lse_out: preallocated contiguous [B, Hq, D]
    and float32 [B, Hq] destinations (lse_out implies the lse is written).
    """
    _check_caches(q, k_cache, v_cache)
    kv_len = _check_len(kv_len, q.shape[0])
    out, lse = _outputs(q, out_dtype, out, lse_out, return_lse)
    a = make_args(q, k_cache, v_cache, kv_len, max_kv_len or 0, sm_scale or 0.0, rotate_q, v_rotated, out, lse,
                  _btype(k_cache), _btype(v_cache))
    lib = _bind()
    need = lib.tq_decode_attention_workspace_size(C.byref(a))
    if need == 0:
        # argument error: let the launch report it with a message
        L.check(lib.tq_decode_attention_cuda(C.byref(a), _stream(q)))
    ws = _workspace(q.device, need)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    L.check(lib.tq_decode_attention_cuda(C.byref(a), _stream(q)))
    return (out, lse) if return_lse else out


def decode_attention_paged(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor,
                           kv_len: torch.Tensor, max_kv_len: int | None = None, sm_scale: float | None = None,
                           rotate_q: bool = True, v_rotated: bool = True, out_dtype: torch.dtype = torch.float32,
                           return_lse: bool = False, out: torch.Tensor | None = None,
                           lse_out: torch.Tensor | None = None):
    """decode_attention over paged caches (tq_decode_attention_paged_cuda).

    k_pool / v_pool: uint8 [num_pages, n_kv_heads, page_size, head_dim/32, bytes];
    page_table: int32 CUDA [B, max_pages_per_seq], row b listing the pool pages of
    sequence b's tokens in order; kv_len: int32 CUDA [B].  Bit-identical to
    decode_attention on the same tokens stored contiguously.
    """
    _check_caches(q, k_pool, v_pool)
    kv_len = _check_len(kv_len, q.shape[0])
    _need_cuda(page_table)
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != q.shape[0] \
            or not page_table.is_contiguous():
        raise ValueError("page_table must be a contiguous int32 [batch, max_pages_per_seq] tensor")
    if k_pool.shape[:3] != v_pool.shape[:3]:
        raise ValueError("K and V pools must have the same pages, heads and page size")
    num_pages, _, page_size = k_pool.shape[:3]
    out, lse = _outputs(q, out_dtype, out, lse_out, return_lse)
    a = make_args(q, k_pool, v_pool, kv_len, max_kv_len or 0, sm_scale or 0.0, rotate_q, v_rotated, out, lse,
                  _btype(k_pool), _btype(v_pool))
    a.kv_capacity = page_table.shape[1] * page_size
    pg = make_pages(page_table, num_pages, page_size)
    lib = _bind()
    need = lib.tq_decode_attention_workspace_size(C.byref(a))
    if need:
        ws = _workspace(q.device, need)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    L.check(lib.tq_decode_attention_paged_cuda(C.byref(a), C.byref(pg), _stream(q)))
    return (out, lse) if return_lse else out


# tq_attention_q8_args (include/leankv_tq.h)
_ATTN_Q8 = struct.Struct("iiiiqPiqqqPiqqqPPPPPPqfiiiPPPN")
_MASK = struct.Struct("Pq")                                        # tq_draft_mask
_WEIGHTS = struct.Struct("iiiiqPiqqqPiPPPPqqfiifPPPPN")            # tq_attention_weights_args


def attention_q8_paged(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                       v_scale: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor,
                       q_len: torch.Tensor | None = None, max_kv_len: int | None = None,
                       sm_scale: float | None = None, causal: bool = True, rotate_q: bool = True,
                       v_rotated: bool = True, out_dtype: torch.dtype | None = None, return_lse: bool = False,
                       out: torch.Tensor | None = None, lse_out: torch.Tensor | None = None,
                       status: torch.Tensor | None = None, tree=None):
    """Attention over 8-bit pages (tq_attention_q8_paged_cuda): one query token per sequence, a few, or prompts.

    q [B, Hq, n, D] of any batch, head and token strides, or [B, Hq, D] for one token; pools int8
    [num_pages, n_kv_heads, page_size, D] with float32 scales [num_pages, n_kv_heads, page_size / 16] as
    ops.kv_append_rotary_paged writes them; page_table int32 [B, max_pages_per_seq]; kv_len int32 [B], the
    cached tokens with this step's.  Query token i of the q_len[b] (default and at most n) of sequence b is cached token
    kv_len[b] - q_len[b] + i and sees the tokens up to itself (causal) or all.  Rows that see nothing, those
    of a padded batch (i >= q_len[b]) among them, give zeros and a log-sum-exp of -inf.  max_kv_len: an upper bound
    of kv_len that sizes the work and, for many rows, the work memory (default: the capacity; up to 1 GiB, or what
    one sequence and head needs): tokens behind it may be left out, with status raised.  sm_scale: None or 0 for
    1 / sqrt(D).  out_dtype: q's by default
    (queries enter the products in 11 bits for a bfloat16 output, in 22 for others; weights in 11: a float32 output is
    exact to about 2e-4 of its norm); out [like q] /
    lse_out (float32 [B, Hq, n]): destinations.  status: int32 CUDA tensor [1], raised to 1 (TQ_ERROR_INVALID_VALUE)
    when a page id outside the pool is met or tokens behind max_kv_len are (they are left out), to 7 (TQ_ERROR_TIMEOUT)
    when a wait inside a kernel ran out (its rows are NaN); without one, last_status() tells.
    tree: the query tokens are nodes of a tree of drafted tokens (ops.draft_tree, or masks of one's own, contiguous int32
    [B or 1, n, ceil(n / 32)]): node i sees the tokens before the nodes and those nodes j < q_len[b] whose bit its mask has.
    """
    device = _device_of(q, k_pool, v_pool, k_scale, v_scale, page_table, kv_len, q_len, out, lse_out, status)
    single = q.dim() == 3
    if single:
        q = q.unsqueeze(2)
        out = out.unsqueeze(2) if out is not None else None
    qs = _check_rows(q, "q")
    B, Hq, n, D = q.shape
    Hkv = k_pool.shape[1] if k_pool.dim() == 4 else 0
    pages, page_size = _check_q8_pools(k_pool, v_pool, k_scale, v_scale, Hkv, D)
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError("n_q_heads must be a multiple of n_kv_heads")
    _check_table(page_table, B)
    _check_lengths(kv_len, B, "kv_len")
    if q_len is not None:
        _check_lengths(q_len, B, "q_len")
    if out is None:
        os = (n * Hq * D, D, Hq * D, 1)
        out = torch.empty_strided((B, Hq, n, D), os, dtype=out_dtype or q.dtype, device=q.device)
    elif out.shape != q.shape or not _own_rows(out) or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError("out must have q's shape, head_dim contiguous, every row its own memory")
    else:
        os = _row_strides(out)
    if out.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {out.dtype}")
    lse = lse_out
    if lse is not None:
        if lse.dtype != torch.float32 or lse.numel() != B * Hq * n or not lse.is_contiguous():
            raise ValueError("lse_out must be a contiguous float32 [B, Hq, n] tensor")
    elif return_lse:
        lse = torch.empty(B, Hq, n, dtype=torch.float32, device=q.device)
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 tensor")
    masks = None
    if tree is not None:
        mask = tree.mask if isinstance(tree, DraftTree) else tree
        _device_of(q, mask)
        words = -(-n // 32)
        if mask.dtype != torch.int32 or mask.dim() != 3 or mask.shape[0] not in (1, B) or mask.shape[1:] != (n, words) \
                or not mask.is_contiguous():
            raise ValueError(f"tree must be a contiguous int32 [{B} or 1, {n}, {words}] tensor of masks")
        if not causal:
            raise ValueError("the rows of a tree are causal")
        masks = _MASK.pack(mask.data_ptr(), 0 if mask.shape[0] == 1 else n * words)
    fields = (B, Hq, Hkv, D, n, q.data_ptr(), _DTYPES[q.dtype], qs[0], qs[1], qs[2], out.data_ptr(), _DTYPES[out.dtype],
              os[0], os[1], os[2], k_pool.data_ptr(), k_scale.data_ptr(), v_pool.data_ptr(), v_scale.data_ptr(),
              kv_len.data_ptr(), 0 if q_len is None else q_len.data_ptr(), int(max_kv_len or 0), float(sm_scale or 0.0),
              int(causal), int(rotate_q), int(v_rotated), 0 if lse is None else lse.data_ptr(),
              0 if status is None else status.data_ptr())
    pg = _PAGES.pack(page_table.data_ptr(), page_table.shape[1], pages, page_size)
    lib = L.load()
    key = ("attention" if masks is None else "tree", device, B, Hq, Hkv, D, n, out.dtype, fields[21], page_table.shape[1], pages, page_size)
    size = lib.tq_attention_q8_workspace_size if masks is None else lib.tq_attention_q8_tree_workspace_size
    need = _work_bytes(key, device, size, _ATTN_Q8, fields, pg)
    # from the allocator on every call: streams and captured graphs each get their own
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    args = _ATTN_Q8.pack(*fields, ws.data_ptr() if need else 0, need)
    if masks is None:
        _call(device, lib.tq_attention_q8_paged_cuda, args, pg)
    else:
        _call(device, lib.tq_attention_q8_tree_paged_cuda, args, pg, masks)
    if single:
        out = out.squeeze(2)
        lse = lse.squeeze(2) if lse is not None and lse.dim() == 3 else lse
    return (out, lse) if return_lse else out


def attention_weights_paged(q: torch.Tensor, k_pool: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor,
                            lse: torch.Tensor, weights: torch.Tensor, k_scale: torch.Tensor | None = None,
                            q_len: torch.Tensor | None = None, fresh: torch.Tensor | None = None, decay: float = 1.0,
                            window: int | None = None, max_kv_len: int | None = None, sm_scale: float | None = None,
                            causal: bool = True, rotate_q: bool = True, status: torch.Tensor | None = None) -> torch.Tensor:
    """Adds up the attention weights that cached tokens get from a step's queries (tq_attention_weights_paged_cuda).

    weights float32 [num_pages, n_kv_heads, page_size], beside the pages: for each token t of sequence b and KV head
    weights <- (t < fresh[b] ? decay * weights : 0) + sum of exp(score - lse) over the group's query heads and those of the last
    `window` (default: all) query tokens that see t.  q, q_len, causal, sm_scale, rotate_q and status as in attention_q8_paged;
    max_kv_len, an upper bound of kv_len, sizes the work split; lse float32 [B, Hq, n] (or [B, Hq] with q [B, Hq, D]), as the
    attention of these queries returned it.
    k_pool: int8 pages with k_scale, or uint8 TQ blocks as decode_attention_paged takes them.  fresh: int32 [B], the first slot
    whose earlier weight is not read (a step's new slots; default: none).  With decay 0 none is read.  Slots behind kv_len keep
    theirs.  Returns weights."""
    device = _device_of(q, k_pool, page_table, kv_len, lse, weights, k_scale, q_len, fresh, status)
    if q.dim() == 3:
        q = q.unsqueeze(2)
    qs = _check_rows(q, "q")
    B, Hq, n, D = q.shape
    pages, H, page_size = _check_weights(weights)
    if H == 0 or Hq == 0 or Hq % H:
        raise ValueError("n_q_heads must be a multiple of n_kv_heads")
    if k_pool.dtype == torch.int8:
        if k_pool.shape != (pages, H, page_size, D) or not k_pool.is_contiguous():
            raise ValueError("8-bit keys must be a contiguous int8 [num_pages, n_kv_heads, page_size, head_dim] tensor, pages as the weights'")
        if k_scale is None or k_scale.dtype != torch.float32 or k_scale.shape != (pages, H, page_size // 16) or not k_scale.is_contiguous():
            raise ValueError("8-bit keys need k_scale, a contiguous float32 [num_pages, n_kv_heads, page_size / 16] tensor")
        kt = L.TYPE_Q8
    else:
        kt = _TYPE_OF_BYTES.get(k_pool.shape[-1])
        if k_pool.dtype != torch.uint8 or kt is None or k_pool.shape != (pages, H, page_size, D // L.QK, L.BLOCK_BYTES[kt]) \
                or not k_pool.is_contiguous():
            raise ValueError("keys must be contiguous uint8 [num_pages, n_kv_heads, page_size, head_dim/32, bytes] blocks, pages as the weights'")
        if k_scale is not None:
            raise ValueError("TQ pools have no scales")
    _check_table(page_table, B)
    _check_lengths(kv_len, B, "kv_len")
    for t, name in ((q_len, "q_len"), (fresh, "fresh")):
        if t is not None:
            _check_lengths(t, B, name)
    if lse.dtype != torch.float32 or lse.numel() != B * Hq * n or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous float32 [B, Hq, n] tensor")
    if window is not None and window < 1:
        raise ValueError("window must be positive")
    p = lambda t: 0 if t is None else t.data_ptr()   # noqa: E731
    fields = (B, Hq, H, D, n, q.data_ptr(), _DTYPES[q.dtype], qs[0], qs[1], qs[2], k_pool.data_ptr(), kt, p(k_scale),
              kv_len.data_ptr(), p(q_len), lse.data_ptr(), int(max_kv_len or 0), int(window or 0), float(sm_scale or 0.0),
              int(causal), int(rotate_q), float(decay), p(fresh), weights.data_ptr(), _check_status(status))
    pg = _PAGES.pack(page_table.data_ptr(), page_table.shape[1], pages, page_size)
    lib = L.load()
    key = ("weights", device, B, Hq, H, D, n, kt, fields[16], fields[17], page_table.shape[1], pages, page_size)
    need = _work_bytes(key, device, lib.tq_attention_weights_workspace_size, _WEIGHTS, fields, pg)
    # from the allocator on every call: streams and captured graphs each get their own
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _call(device, lib.tq_attention_weights_paged_cuda, _WEIGHTS.pack(*fields, ws.data_ptr() if need else 0, need), pg)
    return weights


def _btype(cache: torch.Tensor) -> int:
    return {18: 4, 14: 3, 10: 2}.get(int(cache.shape[-1]), 0)   # 0: rejected by the argument check


def _check_caches(q, k_cache, v_cache) -> None:
    _need_cuda(q, k_cache, v_cache)
    if q.dim() != 3 or not q.is_contiguous():
        raise ValueError("q must be a contiguous [B, Hq, D] tensor")
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise ValueError("caches must be uint8 block tensors")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")


def _check_len(kv_len, batch):
    if kv_len is None:
        return None
    _need_cuda(kv_len)
    if kv_len.dtype != torch.int32 or kv_len.numel() != batch:
        raise ValueError("kv_len must be int32 [batch]")
    return kv_len.contiguous()


def _outputs(q, out_dtype, out, lse_out, return_lse):
    B, Hq, D = q.shape
    if out is None:
        out = torch.empty((B, Hq, D), dtype=out_dtype, device=q.device)
    if lse_out is not None:
        _need_cuda(lse_out)
        if lse_out.dtype != torch.float32 or lse_out.numel() != B * Hq or not lse_out.is_contiguous():
            raise ValueError("lse_out must be a contiguous float32 [B, Hq] tensor")
        return out, lse_out
    return out, (torch.empty((B, Hq), dtype=torch.float32, device=q.device) if return_lse else None)


def last_status(device: torch.device | str | int | None = None) -> int:
    """Kernel-side status on `device` (synchronizes its current stream): that of the last decode_attention, or, if that
    is 0, what attention_q8_paged calls without a status tensor have raised since this was last asked (asking clears it).

    0 (TQ_SUCCESS), 7 (TQ_ERROR_TIMEOUT: a bulk copy or a wait never completed), 2 (TQ_ERROR_UNSUPPORTED: a block
    scale of magnitude >= 2^15) or 1 (TQ_ERROR_INVALID_VALUE: a page id outside the pool, or tokens behind max_kv_len).
    """
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.type == "cuda" and dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    ws = _workspaces.get((dev.type, dev.index))
    status = 0 if ws is None else int(ws[:4].view(torch.int32).item())
    if status == 0:
        word = C.c_int32()
        _call(dev.index, L.load().tq_attention_q8_last_status, C.byref(word))
        status = word.value
    return status


def merge_partials(parts: torch.Tensor, n_parts: int, n_rows: int, head_dim: int, out: torch.Tensor,
                   lse_out: torch.Tensor | None = None) -> torch.Tensor:
    """Log-sum-exp merge of partials packed per part as [o (n_rows*head_dim) | lse (n_rows)] floats.

    parts: contiguous float32 [n_parts * n_rows * (head_dim + 1)] (e.g. the output of
    an all_gather of every rank's packed partial); out: contiguous [n_rows, head_dim]
    of float32/float16/bfloat16 (written); lse_out: optional float32 [n_rows].
    """
    _need_cuda(parts, out)
    stride = n_rows * (head_dim + 1)
    if parts.dtype != torch.float32 or not parts.is_contiguous() or parts.numel() < n_parts * stride:
        raise ValueError("parts must be a contiguous float32 buffer of n_parts packed partials")
    if out.dtype not in _DTYPES or not out.is_contiguous() or out.numel() != n_rows * head_dim:
        raise ValueError("out must be a contiguous [n_rows, head_dim] tensor")
    base = parts.data_ptr()
    L.check(_bind().tq_lse_merge_cuda(n_parts, n_rows, head_dim, base, stride, base + 4 * n_rows * head_dim, stride,
                                      out.data_ptr(), _DTYPES[out.dtype],
                                      lse_out.data_ptr() if lse_out is not None else None, _stream(parts)))
    return out


def lse_combine(o: torch.Tensor, lse: torch.Tensor, return_lse: bool = False):
    """Merge partial results o [P, n, D] (normalized) with natural-log lse [P, n]."""
    _need_cuda(o, lse)
    if o.dtype != torch.float32 or lse.dtype != torch.float32:
        raise ValueError("float32 partials expected")
    o = o.contiguous()
    lse = lse.contiguous()
    P, n, D = o.shape
    out = torch.empty((n, D), dtype=torch.float32, device=o.device)
    lo = torch.empty((n,), dtype=torch.float32, device=o.device) if return_lse else None
    lib = _bind()
    L.check(lib.tq_lse_combine_cuda(P, n, D, o.data_ptr(), lse.data_ptr(), out.data_ptr(),
                                    lo.data_ptr() if lo is not None else None, _stream(o)))
    return (out, lo) if return_lse else out
