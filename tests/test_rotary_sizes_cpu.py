"""Head counts of the rotary and append entry points whose sums pass 32 bits, and block counts whose products pass 64,
are refused (set before any device work)."""
import pytest

from leankv_b200 import _lib as L
from leankv_b200 import ops

MANY = (1 << 31) - 1


def _heads(n, dst=64, src=64):
    return (src, dst, n, 1024, 128, 256, 1024, 128, 256)


@pytest.mark.parametrize("first,second", [(MANY, MANY), (MANY, 1), (1 << 30, 1 << 30), (MANY, None), (1, MANY), ((1 << 24) + 1, None)])
def test_rotary(first, second):
    rope = ops._ROPE.pack(64, 0, 64, 1, 64, 0, 0, 1.0)
    x2 = None if second is None else ops._HEADS.pack(*_heads(second))
    assert L.load().tq_rotary_cuda(rope, 1, 1, 1, 64, ops._HEADS.pack(*_heads(first)), x2, None) == 2


@pytest.mark.parametrize("kv,q", [(1 << 30, 0), (MANY, MANY), (8, MANY), (1 << 24, 0), (8, 1 << 24)])
def test_append(kv, q):
    k = _heads(kv, dst=0)
    a = ops._APPEND.pack(1, kv, 128, 1, 1, *k, *k, *(_heads(q) if q else ops._NO_HEADS), 64, 0, 0, 1, 128, 0, 0, 1.0,
                         64, 8, 64, 64, 8, 64, 0, 0, 1, 0)
    assert L.load().tq_kv_append_rotary_paged_cuda(a, ops._PAGES.pack(64, 4, 8, 16), None) == 2


@pytest.mark.parametrize("blocks", [(1 << 40) + 1, 1 << 57, (1 << 57) + 1, (1 << 63) - 1])
def test_values_of_8_bit_pages(blocks):
    assert L.load().tq_dequantize_q8_cuda(64, 64, 64, 0, blocks, 128, None) == 2
