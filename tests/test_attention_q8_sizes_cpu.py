"""Sizes of attention over 8-bit pages without a device: products that pass 64 bits are refused, and calls that run in
several passes are planned for the pairs of one."""
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


def test_passes_are_planned_for_the_pairs_of_one():
    """72 pairs of 480 rows behind up to 131072 tokens: 1 GiB holds the tiles of 15.  Those have 60 CTAs of 128 rows (30 of
    256) for 148 SMs or so, so their tokens are split, and the work memory has the rows of two splits at least."""
    tokens, pairs = 131072, 15
    tiles = pairs * (tokens // 128) * (4 * 128 * 128 + 128)
    assert tiles <= 1 << 30 < tiles // pairs * (pairs + 1)
    a = _ATTN_Q8.pack(9, 32, 8, 128, 120, 64, 2, 512, 128, 512, 64, 2, 512, 128, 512, 64, 64, 64, 64, 64, 0, 0, 0.0, 1, 1, 1, 0, 0, 0, 0)
    need = L.load().tq_attention_q8_workspace_size(a, ops._PAGES.pack(64, tokens // 16, 8, 16))
    assert need >= tiles + 2 * pairs * 480 * 129 * 4
    # and not those of all 72 pairs
    assert need < tiles + 16 * pairs * 512 * 129 * 4
