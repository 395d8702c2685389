"""Torch-tensor front end of the C ABI (device pointers, current CUDA stream).

Every op requires CUDA tensors and raises otherwise: there is no CPU path.
Packed blocks are uint8 tensors whose last two dims are (n_blocks, 18) for
TQ4_0 or (n_blocks, 14) for TQ3_0 — the byte layout of src/ggml-tq.h:131-141.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from . import _lib as L

QK = L.QK
TQ2_0, TQ3_0, TQ4_0 = L.TYPE_TQ2_0, L.TYPE_TQ3_0, L.TYPE_TQ4_0
Q8, Q8_BLOCK = L.TYPE_Q8, L.Q8_BLOCK
BLOCK_BYTES = L.BLOCK_BYTES
_DTYPES = {torch.float32: L.DTYPE_F32, torch.float16: L.DTYPE_F16, torch.bfloat16: L.DTYPE_BF16}


# the current stream's handle without the Stream object around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)
# the current device, without the lazy-initialization check that a CUDA tensor has made already (0.1 instead of 1 us)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(_raw_stream(t.device.index))


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError("leankv_b200 ops take CUDA tensors only (there is no CPU fallback)")


def _qtype(qtype) -> int:
    q = {2: TQ2_0, 3: TQ3_0, 4: TQ4_0, "tq2_0": TQ2_0, "tq3_0": TQ3_0, "tq4_0": TQ4_0}.get(qtype)
    if q is None:
        raise ValueError(f"unknown TQ type {qtype!r}")
    return q


def quantize(x: torch.Tensor, qtype=4, fwht_head_dim: int = 0, opt_passes: int = 0,
             out: torch.Tensor | None = None, rht_seed: int | None = None, row_len: int | None = None) -> torch.Tensor:
    """[FWHT per fwht_head_dim run] + TQ quantize of a contiguous f32/f16/bf16 tensor.

    Returns uint8 blocks shaped (*x.shape[:-1], x.shape[-1] // 32, block_bytes).
    Bit-exact with hadamard_transform_row + quantize_row_tq*_0_ref
    (src/ggml-tq.c) on x.float(); opt_passes=2 with qtype=3 is LeanKV's TQ3
    optimal rounding (scripts/tq3_rounding.py:74-125).  With rht_seed, every row of
    row_len elements (default: the last dimension) is first rotated as
    randomized_hadamard_transform_row(row, row_len, fwht_head_dim, rht_seed).
    """
    _need_cuda(x)
    q = _qtype(qtype)
    if x.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    if x.shape[-1] % QK:
        raise ValueError("the last dimension must be a multiple of 32")
    shape = (*x.shape[:-1], x.shape[-1] // QK, BLOCK_BYTES[q])
    if out is None:
        out = torch.empty(shape, dtype=torch.uint8, device=x.device)
    else:
        _need_cuda(out)
        if out.dtype != torch.uint8 or out.numel() != x.numel() // QK * BLOCK_BYTES[q] or not out.is_contiguous():
            raise ValueError("out must be a contiguous uint8 tensor of the block size")
    if rht_seed is not None:
        L.check(L.load().tq_quantize_randomized_cuda(q, x.data_ptr(), _DTYPES[x.dtype], out.data_ptr(), x.numel(),
                                                     int(row_len or x.shape[-1]), int(fwht_head_dim),
                                                     int(rht_seed) & 0xFFFFFFFF, int(opt_passes), _stream(x)))
        return out
    L.check(L.load().tq_quantize_cuda(q, x.data_ptr(), _DTYPES[x.dtype], out.data_ptr(), x.numel(),
                                      int(fwht_head_dim), int(opt_passes), _stream(x)))
    return out


def dequantize(blocks: torch.Tensor, qtype=4, dtype: torch.dtype = torch.float32,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """dequantize_row_tq*_0 over uint8 blocks (..., n_blocks, block_bytes) -> (..., n_blocks*32)."""
    _need_cuda(blocks)
    q = _qtype(qtype)
    if blocks.dtype != torch.uint8 or not blocks.is_contiguous():
        raise ValueError("blocks must be a contiguous uint8 tensor")
    bb, held = BLOCK_BYTES[q], blocks.shape
    nb, rest = divmod(blocks.numel(), bb)
    if rest:
        raise ValueError("block buffer size is not a multiple of the block size")
    if len(held) >= 2 and held[-1] == bb:
        shape = (*held[:-2], held[-2] * QK)
    else:
        shape = (nb * QK,)
    if out is None:
        out = torch.empty(*shape, dtype=dtype, device=blocks.device)
    else:
        _need_cuda(out)
        if out.numel() != nb * QK or not out.is_contiguous() or out.dtype not in _DTYPES:
            raise ValueError("bad out tensor")
    L.check(L.load().tq_dequantize_cuda(q, blocks.data_ptr(), out.data_ptr(), _DTYPES[out.dtype], nb * QK,
                                        _stream(blocks)))
    return out


def hadamard_(x: torch.Tensor, head_dim: int) -> torch.Tensor:
    """In-place hadamard_transform_row (src/ggml-tq.c:398-404) on a contiguous float32 tensor."""
    _need_cuda(x)
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("x must be a contiguous float32 tensor")
    L.check(L.load().tq_hadamard_cuda(x.data_ptr(), x.numel(), int(head_dim), _stream(x)))
    return x


def kv_append(src: torch.Tensor, cache: torch.Tensor, pos: torch.Tensor | None = None, qtype=None,
              rotate: bool = True, opt_passes: int = 0, overflow: torch.Tensor | None = None) -> torch.Tensor:
    """Quantize-on-write of new head rows into a packed KV cache (tq_kv_append_cuda).

    src [batch, n_kv_heads, n_new, head_dim] (f32/f16/bf16); cache uint8
    [batch, n_kv_heads, capacity, head_dim/32, block_bytes]; row t of (b, h) lands
    in token slot pos[b] + t (pos: int32 CUDA tensor [batch], None = slot t).
    rotate applies the head_dim Hadamard rotation first.  Slots outside the
    capacity are skipped and counted into overflow (int32 CUDA tensor [1]) when
    given.  Returns cache.
    """
    _need_cuda(src, cache)
    if src.dim() != 4 or not src.is_contiguous() or src.dtype not in _DTYPES:
        raise ValueError("src must be a contiguous f32/f16/bf16 [batch, n_kv_heads, n_new, head_dim] tensor")
    if cache.dim() != 5 or cache.dtype != torch.uint8 or not cache.is_contiguous():
        raise ValueError("cache must be a contiguous uint8 [batch, n_kv_heads, capacity, head_dim/32, bytes] tensor")
    B, H, n_new, D = src.shape
    if qtype is None:
        qtype = TQ4_0 if cache.shape[-1] == BLOCK_BYTES[TQ4_0] else TQ3_0
    q = _qtype(qtype)
    if cache.shape[0] != B or cache.shape[1] != H or cache.shape[3] * QK != D or cache.shape[4] != BLOCK_BYTES[q]:
        raise ValueError(f"cache shape {tuple(cache.shape)} does not match src {tuple(src.shape)} / type {q}")
    if pos is not None:
        _need_cuda(pos)
        if pos.dtype != torch.int32 or pos.numel() != B or not pos.is_contiguous():
            raise ValueError("pos must be a contiguous int32 [batch] tensor")
    if overflow is not None:
        _need_cuda(overflow)
        if overflow.dtype != torch.int32:
            raise ValueError("overflow must be an int32 tensor")
    L.check(L.load().tq_kv_append_cuda(q, src.data_ptr(), _DTYPES[src.dtype], cache.data_ptr(), B, H, D,
                                       cache.shape[2], n_new, pos.data_ptr() if pos is not None else None,
                                       int(rotate), int(opt_passes),
                                       overflow.data_ptr() if overflow is not None else None, _stream(src)))
    return cache


def kv_append_paged(src: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, pos: torch.Tensor | None = None,
                    qtype=None, rotate: bool = True, opt_passes: int = 0,
                    overflow: torch.Tensor | None = None) -> torch.Tensor:
    """kv_append into a paged cache (tq_kv_append_paged_cuda).

    pool uint8 [num_pages, n_kv_heads, page_size, head_dim/32, block_bytes];
    page_table int32 CUDA [batch, max_pages_per_seq]: token slot s of sequence b
    lives in pool page page_table[b, s // page_size] at row s % page_size.  Rows
    whose slot is past max_pages_per_seq * page_size, or whose page id is outside
    the pool, are skipped and counted into overflow.  Returns pool.
    """
    from .attention import make_pages
    _need_cuda(src, pool, page_table)
    if src.dim() != 4 or not src.is_contiguous() or src.dtype not in _DTYPES:
        raise ValueError("src must be a contiguous f32/f16/bf16 [batch, n_kv_heads, n_new, head_dim] tensor")
    if pool.dim() != 5 or pool.dtype != torch.uint8 or not pool.is_contiguous():
        raise ValueError("pool must be a contiguous uint8 [num_pages, n_kv_heads, page_size, head_dim/32, bytes] tensor")
    B, H, n_new, D = src.shape
    if qtype is None:
        qtype = TQ4_0 if pool.shape[-1] == BLOCK_BYTES[TQ4_0] else TQ3_0
    q = _qtype(qtype)
    if pool.shape[1] != H or pool.shape[3] * QK != D or pool.shape[4] != BLOCK_BYTES[q]:
        raise ValueError(f"pool shape {tuple(pool.shape)} does not match src {tuple(src.shape)} / type {q}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B \
            or not page_table.is_contiguous():
        raise ValueError("page_table must be a contiguous int32 [batch, max_pages_per_seq] tensor")
    if pos is not None:
        _need_cuda(pos)
        if pos.dtype != torch.int32 or pos.numel() != B or not pos.is_contiguous():
            raise ValueError("pos must be a contiguous int32 [batch] tensor")
    if overflow is not None:
        _need_cuda(overflow)
        if overflow.dtype != torch.int32:
            raise ValueError("overflow must be an int32 tensor")
    pg = make_pages(page_table, pool.shape[0], pool.shape[2])
    L.check(L.load().tq_kv_append_paged_cuda(q, src.data_ptr(), _DTYPES[src.dtype], pool.data_ptr(), B, H, D,
                                             C.byref(pg), n_new, pos.data_ptr() if pos is not None else None,
                                             int(rotate), int(opt_passes),
                                             overflow.data_ptr() if overflow is not None else None, _stream(src)))
    return pool


# ── rotation by position ─────────────────────────────────────────────────────

class Rotary(NamedTuple):
    """How head rows turn with their positions (tq_rope in include/leankv_tq.h).

    inv_freq: float64 CUDA tensor [rotary_dim / 2], the angle of each pair per position step
    (rotary_frequencies() gives the usual ones; scaling rules come as values).  axis: int32 CUDA tensor
    [rotary_dim / 2], the position axis of each pair (rotary_axes()), None for one axis; entries outside the
    positions' axes take the nearest one (device data, not checked).  Pairs are the elements
    (i, i + rotary_dim / 2), or (2i, 2i + 1) when interleaved; scale, not 0, multiplies the turned part.
    """
    inv_freq: torch.Tensor
    axis: torch.Tensor | None = None
    interleaved: bool = False
    scale: float = 1.0


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """theta^(-2 i / rotary_dim), i = 0 .. rotary_dim / 2 - 1, as float64."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    return (float(theta) ** (-2.0 * i / rotary_dim)).to(device)


def rotary_axes(sections, device="cuda", interleaved: bool = False) -> torch.Tensor:
    """Position axis of each pair, int32: sections[a] pairs turn with axis a, in consecutive runs, or, when
    interleaved, dealt out in turn (pair 0 to axis 0, pair 1 to axis 1, ...) until an axis has its share."""
    left = [int(n) for n in sections]
    if not left or min(left) < 0:
        raise ValueError("sections must be counts of pairs, one per axis")
    if not interleaved:
        return torch.tensor([a for a, n in enumerate(left) for _ in range(n)], dtype=torch.int32, device=device)
    order = []
    while any(left):
        for a, n in enumerate(left):
            if n:
                order.append(a)
                left[a] -= 1
    return torch.tensor(order, dtype=torch.int32, device=device)


# Argument blocks of include/leankv_tq.h as native struct layouts (packing one takes a fraction of the time of
# filling ctypes structures, which is most of a small call).
_ROPE_FMT, _HEADS_FMT = "PPPiiiid", "PPiqqqqqq"
_ROPE = struct.Struct(_ROPE_FMT)                      # tq_rope
_HEADS = struct.Struct(_HEADS_FMT)                    # tq_head_rows
_APPEND = struct.Struct("iiiqi0q" + 3 * _HEADS_FMT + _ROPE_FMT + "PiPPiPPPiP")   # tq_rotary_append_args
_PAGES = struct.Struct("Pqqi")                        # tq_kv_pages
_TYPE_OF_BYTES = {n: t for t, n in BLOCK_BYTES.items()}
_NO_HEADS, _NO_ROPE = (0,) * 9, (0, 0, 0, 0, 0, 0, 0, 0.0)

def _device_of(*ts) -> int:
    """The CUDA device that holds all tensors (None entries are skipped)."""
    d = ts[0].get_device()
    for t in ts:
        if t is not None and (t.get_device() != d or d < 0):
            _need_cuda(*(u for u in ts if u is not None))
            raise ValueError(f"tensors on {ts[0].device} and {t.device}")
    return d


def _on(device: int, fn, *args):
    """A library function with `device` the current one: work is planned for it and launched on it."""
    if device == _current_device():
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


_work_sizes: dict = {}


def _work_bytes(key: tuple, device: int, fn, fmt: struct.Struct, fields: tuple, pg: bytes) -> int:
    """Bytes of work memory of a call, which depend on its sizes and its device (key) alone."""
    n = _work_sizes.get(key)
    if n is None:
        n = _on(device, fn, fmt.pack(*fields, 0, 0), pg)
        if n == 0 and L.load().tq_last_error_string():
            return 0   # arguments that are refused: the call itself says why
        if len(_work_sizes) >= 4096:
            _work_sizes.clear()
        _work_sizes[key] = n
    return n


def _call(device: int, fn, *args) -> None:
    """A library call on the device's current stream."""
    status = _on(device, fn, *args, _raw_stream(device))
    if status:
        L.check(status)


def _row_strides(t: torch.Tensor) -> tuple:
    """Batch, head and token strides; those of dimensions of one, which lead nowhere and may be anything (odd ones would
    be refused as misaligned, unequal ones in place), as a packed tensor has them."""
    B, H, n, D = t.shape
    s = t.stride()
    return (s[0] if B > 1 else 0, s[1] if H > 1 else D, s[2] if n > 1 else 0)


def _check_rows(t: torch.Tensor, name: str) -> tuple:
    """The strides of [batch, heads, tokens, head_dim] rows."""
    s = t.stride()
    if len(s) != 4 or t.dtype not in _DTYPES or (s[3] != 1 and t.shape[3] > 1):
        raise ValueError(f"{name} must be a f32/f16/bf16 [batch, heads, tokens, head_dim] tensor, head_dim contiguous")
    return _row_strides(t) if (s[0] | s[1] | s[2]) & 7 else s   # the usual strides are fine as they are


def _check_lengths(t: torch.Tensor, batch: int, name: str) -> None:
    if t.dtype != torch.int32 or t.numel() != batch or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [batch] tensor")


def _check_table(t: torch.Tensor, batch: int) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != batch or not t.is_contiguous():
        raise ValueError("page_table must be a contiguous int32 [batch, max_pages_per_seq] tensor")


def _check_q8_pools(k_pool, v_pool, k_scale, v_scale, H: int, D: int) -> tuple:
    """(pages, page_size) of 8-bit pools and their scales."""
    shape = k_pool.shape
    if k_pool.dtype != torch.int8 or len(shape) != 4 or shape[1] != H or shape[3] != D or not k_pool.is_contiguous() \
            or v_pool.dtype != torch.int8 or v_pool.shape != shape or not v_pool.is_contiguous():
        raise ValueError("8-bit pools must be contiguous int8 [num_pages, n_kv_heads, page_size, head_dim], both alike")
    want = (shape[0], H, shape[2] // Q8_BLOCK)
    for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if s is None or s.dtype != torch.float32 or s.shape != want or not s.is_contiguous():
            raise ValueError(f"8-bit pools need {name}, a contiguous float32 [num_pages, n_kv_heads, page_size / 16] tensor")
    return shape[0], shape[2]


def _own_rows(t: torch.Tensor) -> bool:
    """head_dim contiguous, and no dimension expanded (rows written over one another)."""
    return all(n <= 1 or (s == 1 if i == 3 else s != 0) for i, (n, s) in enumerate(zip(t.shape, t.stride())))


def _rows_out(t: torch.Tensor, strides: tuple, out: torch.Tensor | None, name: str) -> tuple:
    """The destination of t's rows, and the strides of both (in place: the same ones)."""
    if out is None:
        # token-major memory, as the projections on either side have it
        B, H, n, D = t.shape
        s = (n * H * D, D, H * D, 1)
        return torch.empty_strided((B, H, n, D), s, dtype=t.dtype, device=t.device), strides, s
    if out.shape != t.shape or out.dtype != t.dtype or not _own_rows(out):
        raise ValueError(f"{name} must have the shape and type of its input, head_dim contiguous, every row its own memory")
    return out, _row_strides(t), _row_strides(out)


def _rope_fields(rope: Rotary, batch: int, tokens: int, positions: torch.Tensor | None, inverse: bool) -> tuple:
    """tq_rope's fields, checked (devices apart)."""
    f, ax, interleaved, scale = rope
    if f.dtype != torch.float64 or f.dim() != 1 or not f.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 [rotary_dim / 2] tensor")
    if ax is not None and (ax.dtype != torch.int32 or ax.shape != f.shape or not ax.is_contiguous()):
        raise ValueError("axis must be a contiguous int32 tensor of inv_freq's shape")
    if scale == 0:   # the argument block's 0 stands for 1
        raise ValueError("scale must not be 0")
    axes, where = 1, 0
    if positions is not None:
        shape = positions.shape
        if positions.dtype != torch.int32 or not positions.is_contiguous() or len(shape) not in (2, 3) \
                or shape[-2] != batch or shape[-1] != tokens:
            raise ValueError("positions must be a contiguous int32 [batch, tokens] or [axes, batch, tokens] tensor")
        axes = shape[0] if len(shape) == 3 else 1
        if axes > 1 and ax is None:
            raise ValueError("positions of several axes need the axis of each pair")
        where = positions.data_ptr()
    return (f.data_ptr(), 0 if ax is None else ax.data_ptr(), where, axes, 2 * f.shape[0], int(interleaved), int(inverse),
            float(scale))


def rotary(q: torch.Tensor, positions: torch.Tensor, rope: Rotary, k: torch.Tensor | None = None,
           inverse: bool = False, out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Rotates head rows by their positions (tq_rotary_cuda); q (and k, in the same launch) are
    [batch, heads, tokens, head_dim] of any batch, head and token strides.

    positions: int32 [batch, tokens], or [axes, batch, tokens] with rope.axis naming each pair's axis.
    Computed in float32, rounded once; angles are within 2^-64 turns times the position (3.4e-13 radians at a
    million).  inverse turns back: the gradient of the inputs from that of the outputs.  out / k_out: destinations (may be q / k themselves).
    Returns the rotated q, or (q, k)."""
    if positions is None:
        raise ValueError("positions are needed")
    device = _device_of(q, positions, rope.inv_freq, rope.axis, k, out, k_out)
    qs = _check_rows(q, "q")
    B, H, n, D = q.shape
    r = _rope_fields(rope, B, n, positions, inverse)
    out, qs, os = _rows_out(q, qs, out, "out")
    x = _HEADS.pack(q.data_ptr(), out.data_ptr(), H, qs[0], qs[1], qs[2], os[0], os[1], os[2])
    x2 = None
    if k is not None:
        ks = _check_rows(k, "k")
        if k.dtype != q.dtype or k.shape[0] != B or k.shape[2] != n or k.shape[3] != D:
            raise ValueError("k must have q's type, batch, tokens and head_dim")
        k_out, ks, os = _rows_out(k, ks, k_out, "k_out")
        x2 = _HEADS.pack(k.data_ptr(), k_out.data_ptr(), k.shape[1], ks[0], ks[1], ks[2], os[0], os[1], os[2])
    elif k_out is not None:
        raise ValueError("k_out without k")
    _call(device, L.load().tq_rotary_cuda, _ROPE.pack(*r), _DTYPES[q.dtype], B, n, D, x, x2)
    return out if k is None else (out, k_out)


def kv_append_rotary_paged(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                           page_table: torch.Tensor, pos: torch.Tensor | None = None, rope: Rotary | None = None,
                           positions: torch.Tensor | None = None, q: torch.Tensor | None = None,
                           q_out: torch.Tensor | None = None, new_len: torch.Tensor | None = None,
                           k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                           rotate: bool = True, overflow: torch.Tensor | None = None) -> torch.Tensor | None:
    """A step's rows into a paged cache in one launch (tq_kv_append_rotary_paged_cuda): keys are rotated by
    position and quantized into k_pool, values quantized into v_pool, queries rotated.

    k, v [batch, n_kv_heads, n_new, head_dim] and q [batch, n_q_heads, n_new, head_dim] may have any batch,
    head and token strides (views of one projection's output).  Row t of sequence b goes to slot pos[b] + t
    of its pages.  rope None stores the keys unturned; positions default to the slots.  Pools: uint8 TQ
    blocks as in kv_append_paged (TQ2_0 / TQ3_0 / TQ4_0 keys, TQ4_0 values), or int8
    [num_pages, n_kv_heads, page_size, head_dim] with float32 scales k_scale / v_scale
    [num_pages, n_kv_heads, page_size / 16] (both pools).  new_len (int32 [batch]): rows t >= new_len[b] of
    a padded batch are not stored.  rotate: the head_dim Hadamard rotation, as the attention expects.
    Rows without a place are counted into overflow, keys and values each.  Returns the rotated q (in q_out
    when given, which may be q), or None without q."""
    device = _device_of(k, v, k_pool, v_pool, page_table, pos, new_len, k_scale, v_scale, q, q_out, overflow, positions,
                        *((rope.inv_freq, rope.axis) if rope is not None else ()))
    ks, vs = _check_rows(k, "k"), _check_rows(v, "v")
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("k and v must have the same shape and type")
    B, H, n_new, D = k.shape
    _check_table(page_table, B)
    if k_pool.dtype == torch.int8:
        kt = vt = Q8
        pages, page_size = _check_q8_pools(k_pool, v_pool, k_scale, v_scale, H, D)
        k_sc, v_sc = k_scale.data_ptr(), v_scale.data_ptr()
    else:
        kt, vt = _TYPE_OF_BYTES.get(k_pool.shape[-1]), TQ4_0
        pages, page_size = (k_pool.shape[0], k_pool.shape[2]) if k_pool.dim() == 5 else (0, 0)
        if k_pool.dtype != torch.uint8 or v_pool.dtype != torch.uint8 or kt is None \
                or k_pool.shape != (pages, H, page_size, D // QK, BLOCK_BYTES[kt]) or not k_pool.is_contiguous() \
                or v_pool.shape != (pages, H, page_size, D // QK, BLOCK_BYTES[TQ4_0]) or not v_pool.is_contiguous():
            raise ValueError("pools must be contiguous uint8 [num_pages, n_kv_heads, page_size, head_dim/32, bytes] "
                             "blocks, TQ4_0 for the values")
        if k_scale is not None or v_scale is not None:
            raise ValueError("TQ pools have no scales")
        k_sc = v_sc = 0
    if pos is not None:
        _check_lengths(pos, B, "pos")
    if new_len is not None:
        _check_lengths(new_len, B, "new_len")
    if overflow is not None and (overflow.dtype != torch.int32 or overflow.numel() < 1):
        raise ValueError("overflow must be an int32 tensor")
    if rope is None and (positions is not None or q is not None):
        raise ValueError("positions or q without a rotation")
    r = _NO_ROPE if rope is None else _rope_fields(rope, B, n_new, positions, False)
    heads = _NO_HEADS
    if q is not None:
        qs = _check_rows(q, "q")
        if q.dtype != k.dtype or q.shape[0] != B or q.shape[2] != n_new or q.shape[3] != D or q.shape[1] == 0:
            raise ValueError("q must have k's type, batch, tokens and head_dim")
        q_out, qs, os = _rows_out(q, qs, q_out, "q_out")
        heads = (q.data_ptr(), q_out.data_ptr(), q.shape[1], qs[0], qs[1], qs[2], os[0], os[1], os[2])
    elif q_out is not None:
        raise ValueError("q_out without q")
    a = _APPEND.pack(B, H, D, n_new, _DTYPES[k.dtype], k.data_ptr(), 0, H, ks[0], ks[1], ks[2], 0, 0, 0,
                     v.data_ptr(), 0, H, vs[0], vs[1], vs[2], 0, 0, 0, *heads, *r,
                     k_pool.data_ptr(), kt, k_sc, v_pool.data_ptr(), vt, v_sc, 0 if pos is None else pos.data_ptr(),
                     0 if new_len is None else new_len.data_ptr(), int(rotate), 0 if overflow is None else overflow.data_ptr())
    _call(device, L.load().tq_kv_append_rotary_paged_cuda, a,
          _PAGES.pack(page_table.data_ptr(), page_table.shape[1], pages, page_size))
    return q_out


def dequantize_q8(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Values of 8-bit pages: int8 [..., tokens, head_dim] (tokens a multiple of 16, head_dim 128 or 256)
    times float32 [..., tokens / 16], rounded to dtype."""
    device = _device_of(codes, scale, out)
    shape = codes.shape
    if codes.dtype != torch.int8 or not codes.is_contiguous() or len(shape) < 2 or shape[-2] % Q8_BLOCK:
        raise ValueError("codes must be a contiguous int8 [..., tokens, head_dim] tensor, tokens a multiple of 16")
    blocks = scale.shape
    if scale.dtype != torch.float32 or not scale.is_contiguous() or len(blocks) != len(shape) - 1 \
            or blocks[:-1] != shape[:-2] or blocks[-1] * Q8_BLOCK != shape[-2]:
        raise ValueError("scale must be a contiguous float32 [..., tokens / 16] tensor")
    if out is None:
        if dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {dtype}")
        out = torch.empty_like(codes, dtype=dtype)   # contiguous as the codes are
    elif out.shape != shape or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of the codes' shape")
    kind = _DTYPES.get(out.dtype)
    if kind is None:
        raise TypeError(f"unsupported dtype {out.dtype}")
    _call(device, L.load().tq_dequantize_q8_cuda, codes.data_ptr(), scale.data_ptr(), out.data_ptr(), kind, scale.numel(), shape[-1])
    return out


# ── trees of drafted tokens, eviction ────────────────────────────────────────

class DraftTree(NamedTuple):
    """Trees of drafted tokens as the attention takes them: mask int32 [batch, n, ceil(n / 32)], bit j & 31 of word j >> 5
    set where node i sees node j; depth int32 [batch, n], 0 for a root."""
    mask: torch.Tensor
    depth: torch.Tensor


def draft_tree(parents: torch.Tensor) -> DraftTree:
    """Ancestor masks and depths of trees of drafted tokens (tq_draft_tree_cuda).

    parents: int32 CUDA [batch, n] (or [n], one tree for all sequences) of any batch stride, the parent of each node, which
    comes before it, -1 for children of the cached tokens (other entries that do not come before their node are taken so, too).
    A node sees itself and its ancestors; its position is that of the first token behind the cached ones plus its
    depth.  At most 4096 nodes."""
    device = _device_of(parents)
    if parents.dtype != torch.int32 or parents.dim() not in (1, 2) or (parents.shape[-1] > 1 and parents.stride(-1) != 1):
        raise ValueError("parents must be an int32 [batch, n] or [n] tensor, n contiguous")
    B, n = (1, parents.shape[0]) if parents.dim() == 1 else parents.shape
    mask = torch.empty((B, n, -(-n // 32)), dtype=torch.int32, device=parents.device)
    depth = torch.empty((B, n), dtype=torch.int32, device=parents.device)
    stride = parents.stride(0) if parents.dim() == 2 else 0
    _call(device, L.load().tq_draft_tree_cuda, parents.data_ptr(), stride, B, n, mask.data_ptr(), depth.data_ptr())
    return DraftTree(mask, depth)


_SELECT = struct.Struct("iiPPPqqqqPP")                # tq_select_args
_MOVE = struct.Struct("iiiqPiPPPiPPiPPPqPPPN")        # tq_kv_move_args


def _check_weights(t: torch.Tensor) -> tuple:
    """(pages, heads, page_size) of a pool of summed attention weights."""
    if t.dtype != torch.float32 or t.dim() != 3 or not t.is_contiguous():
        raise ValueError("weights must be a contiguous float32 [num_pages, n_kv_heads, page_size] tensor")
    return t.shape


def _check_status(t: torch.Tensor | None, name: str = "status") -> int:
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.numel() < 1:
        raise ValueError(f"{name} must be an int32 tensor")
    return t.data_ptr()


def select_tokens(weights: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor, keep, sinks: int = 0,
                  recent: int = 0, width: int | None = None, max_kv_len: int | None = None,
                  out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """The cached tokens of each (sequence, KV head) that stay (tq_select_tokens_cuda).

    weights float32 [num_pages, n_kv_heads, page_size], the sums that attention_weights_paged keeps; page_table int32
    [B, max_pages_per_seq]; kv_len int32 [B].  keep: one number, or int32 CUDA [B] with width, their bound.  Of
    k = min(keep, kv_len, width) tokens the last min(recent, k) stay, the first min(sinks, k - recent), and of the others
    those with the largest weights, ties to the lowest slot, NaN as -inf.  Returns int32 [B, n_kv_heads, width] (in out; with one
    number, keep or the smaller width): slots, rising, -1 behind the last.  max_kv_len: an upper bound of kv_len that sizes the
    work (default: the capacity); tokens behind it are left out, with status raised, as for pages outside the pool
    (attention.last_status() without status)."""
    by_sequence = isinstance(keep, torch.Tensor)
    device = _device_of(weights, page_table, kv_len, out, status, keep if by_sequence else None)
    pages, H, page_size = _check_weights(weights)
    B, per = page_table.shape if page_table.dim() == 2 else (0, 0)
    _check_table(page_table, B)
    _check_lengths(kv_len, B, "kv_len")
    if by_sequence:
        _check_lengths(keep, B, "keep")
        if width is None:
            raise ValueError("a tensor of numbers to keep needs width, their bound")
        each = keep.data_ptr()
    else:
        if int(keep) < 0:
            raise ValueError("keep must not be negative")
        width, each = min(int(keep), int(keep) if width is None else int(width)), 0
    if out is None:
        out = torch.empty(B, H, width, dtype=torch.int32, device=weights.device)
    elif out.dtype != torch.int32 or out.shape != (B, H, width) or not out.is_contiguous():
        raise ValueError("out must be a contiguous int32 [B, n_kv_heads, width] tensor")
    a = _SELECT.pack(B, H, weights.data_ptr(), kv_len.data_ptr(), each, width, int(sinks), int(recent), int(max_kv_len or 0),
                     out.data_ptr(), _check_status(status))
    _call(device, L.load().tq_select_tokens_cuda, a, _PAGES.pack(page_table.data_ptr(), per, pages, page_size))
    return out


def kv_move_paged(k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor, src: torch.Tensor,
                  first: torch.Tensor | None = None, count: torch.Tensor | None = None,
                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                  weights: torch.Tensor | None = None, to_table: torch.Tensor | None = None,
                  overflow: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Moves rows of a paged cache between token slots (tq_kv_move_paged_cuda): the accepted path of a drafted tree, the
    tokens that stay after an eviction.

    Row j of sequence b and KV head h goes from slot src[b, h, j] to slot first[b] + j (first: int32 [B], default 0).  src
    int32 [B, n_kv_heads, n] or, for all heads alike, [B, n]; negative entries move nothing; rows j >= count[b] (int32
    [B]) neither.  Pools as kv_append_rotary_paged writes them (TQ rows are copied; 8-bit blocks of rows of one scale keep
    codes and scale, others get max |code| scale / 127).  weights: pool of summed attention weights, moved along.  In place
    (no to_table, or page_table itself) rows may only move down (src >= first + j); another to_table (int32 [B, pages]) names
    other pages for the destination, none that are read.  Rows without a place, or that would move up, are left and counted into
    overflow, one per head."""
    device = _device_of(k_pool, v_pool, page_table, src, first, count, k_scale, v_scale, weights, to_table, overflow, status)
    B = page_table.shape[0]
    _check_table(page_table, B)
    if k_pool.dtype == torch.int8:
        H, D = (k_pool.shape[1], k_pool.shape[3]) if k_pool.dim() == 4 else (0, 0)
        pages, page_size = _check_q8_pools(k_pool, v_pool, k_scale, v_scale, H, D)
        kt = vt = Q8
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    else:
        if k_pool.dim() != 5 or v_pool.dim() != 5 or k_pool.dtype != torch.uint8 or v_pool.dtype != torch.uint8 \
                or k_pool.shape[:4] != v_pool.shape[:4] or v_pool.shape[4] != BLOCK_BYTES[TQ4_0] \
                or k_pool.shape[4] not in _TYPE_OF_BYTES or not k_pool.is_contiguous() or not v_pool.is_contiguous():
            raise ValueError("pools must be contiguous uint8 [num_pages, n_kv_heads, page_size, head_dim/32, bytes] "
                             "blocks, TQ4_0 for the values")
        if k_scale is not None or v_scale is not None:
            raise ValueError("TQ pools have no scales")
        pages, H, page_size, D = k_pool.shape[0], k_pool.shape[1], k_pool.shape[2], k_pool.shape[3] * QK
        kt, vt, ks, vs = _TYPE_OF_BYTES[k_pool.shape[4]], TQ4_0, 0, 0
    if src.dtype != torch.int32 or src.dim() not in (2, 3) or src.shape[0] != B or not src.is_contiguous() \
            or (src.dim() == 3 and src.shape[1] not in (1, H)):
        raise ValueError("src must be a contiguous int32 [B, n_kv_heads, n] or [B, n] tensor")
    for t, name in ((first, "first"), (count, "count")):
        if t is not None:
            _check_lengths(t, B, name)
    if weights is not None and _check_weights(weights) != (pages, H, page_size):
        raise ValueError(f"weights must be [{pages}, {H}, {page_size}], as the pools")
    if to_table is not None:
        _check_table(to_table, B)
        if to_table.shape[1] == 0:
            raise ValueError("to_table must have a page for each sequence at least")   # (without one its address is that of no table)
    rows, per = src.shape[-1], page_table.shape[1]
    fields = (B, H, D, rows, src.data_ptr(), src.shape[1] if src.dim() == 3 else 1, 0 if first is None else first.data_ptr(),
              0 if count is None else count.data_ptr(), k_pool.data_ptr(), kt, ks, v_pool.data_ptr(), vt, vs,
              0 if weights is None else weights.data_ptr(), 0 if to_table is None else to_table.data_ptr(),
              0 if to_table is None else to_table.shape[1], _check_status(overflow, "overflow"), _check_status(status))
    pg = _PAGES.pack(page_table.data_ptr(), per, pages, page_size)
    lib = L.load()
    # a table of the destinations that is the pages' own is in place, too
    in_place = to_table is None or to_table.data_ptr() == page_table.data_ptr()
    key = ("move", device, B, H, D, rows, kt, first is None, in_place, per, pages, page_size)
    need = _work_bytes(key, device, lib.tq_kv_move_workspace_size, _MOVE, fields, pg)
    # from the allocator on every call: streams and captured graphs each get their own
    ws = torch.empty(need, dtype=torch.uint8, device=k_pool.device) if need else None
    _call(device, lib.tq_kv_move_paged_cuda, _MOVE.pack(*fields, ws.data_ptr() if need else 0, need), pg)


TQ2_1_BYTES = 44   # block_tq2_1: a TQ3_0 block and three TQ2_0 blocks per 128 elements


def quantize_tq2_1(x: torch.Tensor) -> torch.Tensor:
    """TQ2_1 blocks (the fork's static mixed-precision type, tq_quantize_tq2_1_cuda) of a contiguous
    f32/f16/bf16 tensor whose last dim is a multiple of 128: uint8 (..., last / 128, 44).  No
    rotation is applied (rotate first with hadamard_ when the rows should be rotated)."""
    _need_cuda(x)
    if x.dtype not in _DTYPES or not x.is_contiguous() or x.dim() == 0 or x.shape[-1] % 128:
        raise ValueError("x must be a contiguous f32/f16/bf16 tensor whose last dim is a multiple of 128")
    out = torch.empty((*x.shape[:-1], x.shape[-1] // 128, TQ2_1_BYTES), dtype=torch.uint8, device=x.device)
    L.check(L.load().tq_quantize_tq2_1_cuda(x.data_ptr(), _DTYPES[x.dtype], out.data_ptr(), x.numel(), _stream(x)))
    return out


def dequantize_tq2_1(blocks: torch.Tensor) -> torch.Tensor:
    """float32 (..., n_blocks * 128) from uint8 TQ2_1 blocks (..., n_blocks, 44)."""
    _need_cuda(blocks)
    if blocks.dtype != torch.uint8 or not blocks.is_contiguous() or blocks.dim() < 2 \
            or blocks.shape[-1] != TQ2_1_BYTES:
        raise ValueError("blocks must be a contiguous uint8 (..., n_blocks, 44) tensor")
    out = torch.empty((*blocks.shape[:-2], blocks.shape[-2] * 128), dtype=torch.float32, device=blocks.device)
    L.check(L.load().tq_dequantize_tq2_1_cuda(blocks.data_ptr(), out.data_ptr(), out.numel(), _stream(blocks)))
    return out


def requantize(blocks: torch.Tensor, src_qtype, dst_qtype) -> torch.Tensor:
    """Blocks of src_qtype -> blocks of dst_qtype (dequantize + quantize per block, one kernel;
    requantize_tq4_to_tq3 / tq3_to_tq2 / tq4_to_tq2 of src/ggml-tq.c:329-357)."""
    _need_cuda(blocks)
    a, b = _qtype(src_qtype), _qtype(dst_qtype)
    if blocks.dtype != torch.uint8 or not blocks.is_contiguous() or blocks.numel() % BLOCK_BYTES[a]:
        raise ValueError("blocks must be a contiguous uint8 tensor of whole blocks")
    nb = blocks.numel() // BLOCK_BYTES[a]
    shape = (*blocks.shape[:-1], BLOCK_BYTES[b]) if blocks.dim() >= 1 and blocks.shape[-1] == BLOCK_BYTES[a] \
        else (nb, BLOCK_BYTES[b])
    out = torch.empty(shape, dtype=torch.uint8, device=blocks.device)
    L.check(L.load().tq_requantize_cuda(a, blocks.data_ptr(), b, out.data_ptr(), nb * QK, _stream(blocks)))
    return out


def hadamard_randomized_(x: torch.Tensor, head_dim: int, seed: int, row_len: int | None = None) -> torch.Tensor:
    """In-place randomized_hadamard_transform_row (src/ggml-tq.c:383-412) on every row of row_len
    elements (default: the last dimension) of a contiguous float32 tensor."""
    _need_cuda(x)
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("x must be a contiguous float32 tensor")
    L.check(L.load().tq_hadamard_randomized_cuda(x.data_ptr(), x.numel(), int(row_len or x.shape[-1]), int(head_dim),
                                                 int(seed) & 0xFFFFFFFF, _stream(x)))
    return x


class OutlierConfig(C.Structure):
    """Mirror of tq_outlier_config (src/ggml-tq-outlier.h:44-64, include/leankv_tq.h)."""
    _fields_ = [("head_dim", C.c_int), ("n_outlier", C.c_int), ("n_normal", C.c_int), ("outlier_frac", C.c_float),
                ("outlier_tier", C.c_int), ("normal_tier", C.c_int), ("perm", C.c_int * 256),
                ("inv_perm", C.c_int * 256), ("channel_var", C.c_float * 256)]


TIER_TQ2, TIER_TQ3, TIER_TQ4 = 0, 1, 2
_TIER_BYTES = {TIER_TQ2: 10, TIER_TQ3: 14, TIER_TQ4: 18}


def identify_outliers(calib: torch.Tensor, outlier_frac: float = 0.25, outlier_tier: int = TIER_TQ3,
                      normal_tier: int = TIER_TQ2) -> OutlierConfig:
    """Per-channel variance ranking of calibration data [n_tokens, head_dim] (float32, CUDA)
    -> outlier configuration (tq_identify_outliers, src/ggml-tq-outlier.c:97-170)."""
    _need_cuda(calib)
    if calib.dtype != torch.float32 or calib.dim() != 2 or not calib.is_contiguous():
        raise ValueError("calib must be a contiguous float32 [n_tokens, head_dim] tensor")
    cfg = OutlierConfig()
    L.check(L.load().tq_outlier_identify_cuda(C.byref(cfg), calib.data_ptr(), calib.shape[0], calib.shape[1],
                                              float(outlier_frac), int(outlier_tier), int(normal_tier), _stream(calib)))
    return cfg


def mixed_quantize(x: torch.Tensor, cfg: OutlierConfig) -> tuple[torch.Tensor, torch.Tensor]:
    """Channel-permuted two-tier quantization of head vectors x [..., head_dim]
    (tq_mixed_quantize per vector) -> (outlier blocks, normal blocks) uint8."""
    _need_cuda(x)
    if x.dtype not in _DTYPES or not x.is_contiguous() or x.shape[-1] != cfg.head_dim:
        raise ValueError("x must be a contiguous f32/f16/bf16 tensor with head_dim last")
    n_vec = x.numel() // cfg.head_dim
    ob = torch.empty(*x.shape[:-1], cfg.n_outlier // QK, _TIER_BYTES[cfg.outlier_tier], dtype=torch.uint8, device=x.device)
    nb = torch.empty(*x.shape[:-1], cfg.n_normal // QK, _TIER_BYTES[cfg.normal_tier], dtype=torch.uint8, device=x.device)
    L.check(L.load().tq_mixed_quantize_cuda(C.byref(cfg), x.data_ptr(), _DTYPES[x.dtype], n_vec, ob.data_ptr(),
                                            nb.data_ptr(), _stream(x)))
    return ob, nb


def mixed_dequantize(outlier_blocks: torch.Tensor, normal_blocks: torch.Tensor, cfg: OutlierConfig) -> torch.Tensor:
    """Inverse of mixed_quantize: float32 [..., head_dim] in the original channel order."""
    _need_cuda(outlier_blocks, normal_blocks)
    lead = outlier_blocks.shape[:-2] if cfg.n_outlier else normal_blocks.shape[:-2]
    n_vec = 1
    for s in lead:
        n_vec *= s
    y = torch.empty(*lead, cfg.head_dim, dtype=torch.float32, device=outlier_blocks.device)
    L.check(L.load().tq_mixed_dequantize_cuda(C.byref(cfg), outlier_blocks.contiguous().data_ptr(),
                                              normal_blocks.contiguous().data_ptr(), n_vec, y.data_ptr(),
                                              _stream(outlier_blocks)))
    return y
