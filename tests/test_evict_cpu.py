"""Trees of drafted tokens and eviction without a device: what the C entry points refuse, and the page bookkeeping."""
import ctypes as C

import numpy as np
import pytest

from leankv_b200 import _lib as L
from leankv_b200 import ops
from leankv_b200.attention import _ATTN_Q8, _MASK, _WEIGHTS
from leankv_b200.paged import NO_PAGE, PageTable

PAGES = (64, 8, 8, 16)     # table, pages a sequence, pages, page size
INVALID, UNSUPPORTED, MISALIGNED = 1, 2, 3


def _pack(fmt, fields, change):
    return fmt.pack(*{**fields, **change}.values())


def _weights(pages=PAGES, **change):
    a = dict(B=1, Hq=4, H=2, D=128, n=3, q=64, qt=0, q0=1536, q1=128, q2=512, k=64, kt=8, ks=64, kv_len=64, q_len=0, lse=64, most=0, window=0,
             sm=0.0, causal=1, rotate=1, decay=1.0, fresh=0, w=64, status=64, ws=0, bytes=0)
    return L.load().tq_attention_weights_paged_cuda(_pack(_WEIGHTS, a, change), ops._PAGES.pack(*pages), None)


def _select(pages=PAGES, **change):
    a = dict(B=1, H=2, w=64, kv_len=64, keep=0, width=4, sinks=0, recent=0, most=0, out=64, status=64)
    return L.load().tq_select_tokens_cuda(_pack(ops._SELECT, a, change), ops._PAGES.pack(*pages), None)


def _move(pages=PAGES, **change):
    a = dict(B=1, H=2, D=128, n=3, src=64, heads=2, first=0, count=0, k=64, kt=8, ks=64, v=64, vt=8, vs=64, w=0, to=0, to_pages=0, over=0,
             status=64, ws=0, bytes=0)
    return L.load().tq_kv_move_paged_cuda(_pack(ops._MOVE, a, change), ops._PAGES.pack(*pages), None)


@pytest.mark.parametrize("want,change", [
    (INVALID, dict(q=0)), (INVALID, dict(k=0)), (INVALID, dict(ks=0)), (INVALID, dict(lse=0)), (INVALID, dict(kv_len=0)), (INVALID, dict(w=0)),
    (INVALID, dict(B=-1)), (INVALID, dict(Hq=3)), (INVALID, dict(H=0)), (INVALID, dict(n=-1)), (INVALID, dict(most=129)), (INVALID, dict(window=-1)),
    (INVALID, dict(sm=float("nan"))), (INVALID, dict(decay=float("inf"))), (INVALID, dict(qt=7)), (UNSUPPORTED, dict(D=64)),
    (UNSUPPORTED, dict(kt=5)), (UNSUPPORTED, dict(n=1 << 31)), (UNSUPPORTED, dict(n=1 << 62)), (UNSUPPORTED, dict(B=1 << 30)),
    (MISALIGNED, dict(q=68)), (MISALIGNED, dict(q1=127)), (MISALIGNED, dict(k=72)), (MISALIGNED, dict(w=66)), (MISALIGNED, dict(w=72)), (MISALIGNED, dict(lse=65)),
    (INVALID, dict(pages=(0, 8, 8, 16))), (INVALID, dict(pages=(64, 8, 8, 24))), (UNSUPPORTED, dict(pages=(64, 1 << 30, 8, 16)))])
def test_weights_refusals(want, change):
    assert _weights(**change) == want


@pytest.mark.parametrize("want,change", [
    (INVALID, dict(w=0)), (INVALID, dict(kv_len=0)), (INVALID, dict(out=0)), (INVALID, dict(width=-1)), (INVALID, dict(sinks=-1)),
    (INVALID, dict(recent=-1)), (INVALID, dict(most=129)), (INVALID, dict(H=0)), (INVALID, dict(B=-1)), (UNSUPPORTED, dict(width=1 << 31)),
    (UNSUPPORTED, dict(B=1 << 30)), (MISALIGNED, dict(w=66)), (MISALIGNED, dict(w=72)), (MISALIGNED, dict(keep=65)), (INVALID, dict(pages=(64, 0, 8, 16)))])
def test_select_refusals(want, change):
    assert _select(**change) == want


@pytest.mark.parametrize("want,change", [
    (INVALID, dict(src=0)), (INVALID, dict(k=0)), (INVALID, dict(v=0)), (INVALID, dict(ks=0)), (INVALID, dict(vs=0)), (INVALID, dict(n=-1)),
    (INVALID, dict(heads=3)), (INVALID, dict(H=0)), (INVALID, dict(B=-1)), (UNSUPPORTED, dict(D=64)), (UNSUPPORTED, dict(kt=4)),
    (UNSUPPORTED, dict(kt=3, vt=3)), (UNSUPPORTED, dict(n=1 << 31)), (UNSUPPORTED, dict(B=1 << 30, n=1 << 20)), (UNSUPPORTED, dict(to=64, to_pages=1 << 30)),
    (MISALIGNED, dict(k=72)), (MISALIGNED, dict(src=66)), (MISALIGNED, dict(w=65)), (MISALIGNED, dict(first=66)), (INVALID, dict(n=200)),
    (MISALIGNED, dict(n=200, ws=66, bytes=1 << 20)), (INVALID, dict(n=200, ws=64, bytes=8))])
def test_move_refusals(want, change):
    assert _move(**change) == want


def test_move_work_memory_is_for_chunks_in_place():
    size = lambda **c: L.load().tq_kv_move_workspace_size(_pack(ops._MOVE, dict(   # noqa: E731
        B=2, H=2, D=128, n=3, src=64, heads=2, first=0, count=0, k=64, kt=8, ks=64, v=64, vt=8, vs=64, w=0, to=0, to_pages=0, over=0, status=64,
        ws=0, bytes=0), c), ops._PAGES.pack(*PAGES))
    assert size(n=64) == 0 and size(n=65) == 4 * (4 * 2 + 1)
    assert size(n=50, first=64) == 4 * (4 * 2 + 1)     # 50 rows behind up to 15 of the first block
    assert size(n=5000, to=128, to_pages=8) == 0 and size(n=0) == 0


def test_tree_refusals():
    lib = L.load()
    tree = lambda p=64, stride=5, B=1, n=5, m=64, d=64: lib.tq_draft_tree_cuda(p, stride, B, n, m, d, None)   # noqa: E731
    assert tree(p=0) == INVALID and tree(n=-1) == INVALID and tree(B=-1) == INVALID
    assert tree(n=4097) == UNSUPPORTED and tree(B=65536) == UNSUPPORTED and tree(p=66) == MISALIGNED
    assert tree(n=0) == 0 and tree(B=0) == 0 and tree(m=0, d=0) == 0
    args = lambda causal=1: _ATTN_Q8.pack(1, 4, 2, 128, 3, 64, 1, 1536, 128, 512, 64, 1, 1536, 128, 512, 64, 64, 64, 64, 64, 0, 0, 0.0,   # noqa: E731
                                          causal, 1, 1, 0, 64, 0, 0)
    pages = ops._PAGES.pack(*PAGES)
    call = lambda a, m: lib.tq_attention_q8_tree_paged_cuda(a, pages, m, None)   # noqa: E731
    assert call(args(), None) == INVALID and call(args(), _MASK.pack(0, 0)) == INVALID
    assert call(args(causal=0), _MASK.pack(64, 0)) == INVALID and call(args(), _MASK.pack(66, 0)) == MISALIGNED


def test_tree_work_memory_at_the_largest_sizes():
    """Rows and tokens whose products pass 64 bits are planned for all the same."""
    lib = L.load()
    args = lambda B, n: _ATTN_Q8.pack(B, 4, 2, 128, n, 64, 1, 1536, 128, 512, 64, 1, 1536, 128, 512, 64, 64, 64, 64, 64, 0, 0, 0.0,   # noqa: E731
                                      1, 1, 1, 0, 64, 0, 0)
    pages = ops._PAGES.pack(64, 1 << 26, 8, 16)
    for B, n in ((1, 1 << 29), (1 << 29, 1), (1 << 20, 1 << 18)):
        need = lib.tq_attention_q8_tree_workspace_size(args(B, n), pages)
        assert lib.tq_last_error_string() == b"" and need < 1 << 63


def test_truncated_sequences_give_pages_back_and_keep_count():
    pt = PageTable(num_pages=10, page_size=16, max_seqs=2, max_pages_per_seq=8)
    a, b = pt.add_sequence(), pt.add_sequence()
    pt.reserve([a, b], [100, 20])
    pt.commit([a, b], [100, 20])
    held = list(pt.table[a, :7])
    pt.dirty.clear()
    pt.truncate(a, 33)
    assert pt.lens[a] == 33 and pt.dropped[a] == 67 and pt.n_pages[a] == 3 and pt.free_pages == 5 and pt.dirty == {a}
    assert list(pt.table[a, :3]) == held[:3] and (pt.table[a, 3:] == NO_PAGE).all()
    pt.reserve([a], 16)
    assert pt.table[a, 3] == held[3]                   # the pages come back in their order
    pt.truncate(a, 33)
    assert pt.dropped[a] == 67 and pt.n_pages[a] == 3  # reserved ones return, too
    pt.truncate(b, 0)
    assert pt.n_pages[b] == 0 and pt.dropped[b] == 20
    with pytest.raises(ValueError):
        pt.truncate(a, 34)
    pt.free_sequence(a)
    assert pt.dropped[pt.add_sequence()] == 0
    assert isinstance(pt.dropped, np.ndarray)


def test_argument_blocks_have_the_header_s_sizes():
    """struct layouts against what a C compiler makes of include/leankv_tq.h's fields in order."""
    class W(C.Structure):
        _fields_ = [("i", C.c_int * 4), ("n", C.c_int64), ("q", C.c_void_p), ("qt", C.c_int), ("qs", C.c_int64 * 3), ("k", C.c_void_p),
                    ("kt", C.c_int), ("p", C.c_void_p * 4), ("m", C.c_int64 * 2), ("sm", C.c_float), ("c", C.c_int * 2), ("d", C.c_float),
                    ("r", C.c_void_p * 4), ("b", C.c_size_t)]

    class M(C.Structure):
        _fields_ = [("i", C.c_int * 3), ("n", C.c_int64), ("src", C.c_void_p), ("h", C.c_int), ("p", C.c_void_p * 2), ("k", C.c_void_p),
                    ("kt", C.c_int), ("ks", C.c_void_p), ("v", C.c_void_p), ("vt", C.c_int), ("r", C.c_void_p * 3), ("to", C.c_int64),
                    ("e", C.c_void_p * 3), ("b", C.c_size_t)]

    class S(C.Structure):
        _fields_ = [("i", C.c_int * 2), ("p", C.c_void_p * 3), ("n", C.c_int64 * 4), ("o", C.c_void_p * 2)]

    assert (_WEIGHTS.size, ops._MOVE.size, ops._SELECT.size, _MASK.size) == (C.sizeof(W), C.sizeof(M), C.sizeof(S), 16)


class _Library:
    """Plans by the current device; a launch refuses work memory of another device's plan, as the library does."""

    def __init__(self, current):
        self.current, self.seen = current, []

    def _size(self, *_):
        self.seen.append(("size", self.current[0]))
        return {0: 1 << 10, 1: 1 << 12}[self.current[0]]

    def _launch(self, fmt):
        def call(args, *rest):
            self.seen.append(("launch", self.current[0], rest[-1]))
            return 0 if fmt is None or fmt.unpack(args)[-1] >= {0: 1 << 10, 1: 1 << 12}[self.current[0]] else 1
        return call

    tq_attention_weights_workspace_size = tq_kv_move_workspace_size = tq_attention_q8_tree_workspace_size = _size
    tq_attention_weights_paged_cuda = property(lambda self: self._launch(_WEIGHTS))
    tq_kv_move_paged_cuda = property(lambda self: self._launch(ops._MOVE))
    tq_attention_q8_tree_paged_cuda = property(lambda self: self._launch(_ATTN_Q8))
    tq_select_tokens_cuda = property(lambda self: self._launch(None))

    @staticmethod
    def tq_last_error_string():
        return b"workspace too small"


def test_calls_of_tensors_on_another_device(monkeypatch):
    """Work memory is sized, and work launched, on the tensors' device and its stream."""
    import contextlib

    import torch

    from leankv_b200 import attention
    current = [0]
    lib = _Library(current)

    @contextlib.contextmanager
    def guard(device):
        before, current[0] = current[0], device
        yield
        current[0] = before

    for module in (attention, ops):
        monkeypatch.setattr(module, "_device_of", lambda *ts: 1)
    monkeypatch.setattr(L, "load", lambda: lib)
    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 100 + device)
    monkeypatch.setattr(ops, "_work_sizes", {})
    monkeypatch.setattr(torch.cuda, "device", guard)
    pool, scale, w = torch.zeros(4, 1, 16, 128, dtype=torch.int8), torch.zeros(4, 1, 1), torch.zeros(4, 1, 16)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q, src = torch.zeros(1, 2, 3, 128), torch.zeros(1, 1, 40, dtype=torch.int32)
    both = [("size", 1), ("launch", 1, 101)]
    attention.attention_weights_paged(q, pool, table, lens, torch.zeros(1, 2, 3), w, k_scale=scale)
    assert lib.seen == both
    lib.seen.clear()
    ops.kv_move_paged(pool, pool, table, src, k_scale=scale, v_scale=scale)
    assert lib.seen == both
    lib.seen.clear()
    ops.select_tokens(w, table, lens, 4)
    assert lib.seen == both[1:] and current == [0]
