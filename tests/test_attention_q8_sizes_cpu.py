"""Sizes of attention over 8-bit pages whose products pass 64 bits are refused (set before any device work)."""
import pytest

from leankv_b200 import _lib as L
from leankv_b200 import ops
from leankv_b200.attention import _ATTN_Q8


def _call(batch=1, hq=4, hkv=2, n=1, max_pages=64):
    # no query pointer: sizes that are let through end at that
    a = _ATTN_Q8.pack(batch, hq, hkv, 128, n, 0, 1, 512, 128, 512, 64, 1, 512, 128, 512, 64, 64, 64, 64, 64, 0, 0, 0.0, 1, 1, 1, 0, 0,
                      0, 0)
    pages = ops._PAGES.pack(64, max_pages, 8, 16)
    lib = L.load()
    return lib.tq_attention_q8_paged_cuda(a, pages, None), lib.tq_attention_q8_workspace_size(a, pages)


@pytest.mark.parametrize("sizes", [
    dict(hq=8, n=1 << 62),                                    # n * 4 is 2^64
    dict(hq=4, n=(1 << 63) - 1),                              # the largest number
    dict(n=1 << 31), dict(n=(1 << 32) + 1),
    dict(batch=(1 << 31) - 1, hq=(1 << 31) - 2, hkv=2),       # 2^62 rows, 2^31 to a head
    dict(batch=(1 << 31) - 1, hq=(1 << 31) - 1, hkv=(1 << 31) - 1, n=64),
    dict(batch=1 << 20, hq=1 << 20, hkv=1 << 20, n=1)])       # 2^40 pairs
def test_products_past_64_bits(sizes):
    assert _call(**sizes) == (2, 0)


def test_large_sizes_that_fit_go_on():
    assert _call(batch=1 << 20, hq=32, hkv=8, n=1)[0] == 1
    assert _call(batch=1, hq=1, hkv=1, n=1 << 30)[0] == 1
