"""Sums of attention weights of many rows over 8-bit keys (the tcgen05 kernel): rows that see no token, and the rounding of scores."""
import math

import pytest
import torch

from leankv_b200 import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D,grp,n,L,uncounted", [(128, 1, 420, 400, 140), (128, 1, 700, 300, 128), (128, 2, 300, 290, 100), (256, 1, 150, 140, 100),
                                                (128, 8, 20, 12, 3), (128, 1, 20, 12, 3)])
def test_rows_before_the_cache_s_first_token_add_nothing(D, grp, n, L, uncounted):
    """More query rows than cached tokens: the first ones see no token, and what lies in their place of q and lse does not count.  The
    rows behind them, which see the first few tokens, are left out, too (-inf), so that whole tiles of tokens lie before all that the
    counted rows end at."""
    H, P = 2, 16
    g = torch.Generator(device=DEV).manual_seed(n)
    pool = torch.randint(-127, 128, (32, H, P, D), dtype=torch.int8, device=DEV, generator=g)
    scale = torch.rand(32, H, 1, device=DEV, generator=g) / 60
    table = torch.randperm(32, generator=torch.Generator().manual_seed(n))[:26].to(torch.int32).view(1, 26).to(DEV)
    lens = torch.tensor([L], dtype=torch.int32, device=DEV)
    q = torch.randn(1, H * grp, n, D, device=DEV, generator=g)
    lse = torch.full((1, H * grp, n), 4.0, device=DEV)
    lse[:, :, n - L: n - L + uncounted] = -math.inf
    blind, other = lse.clone(), q.clone()
    blind[:, :, : n - L] = -math.inf
    other[:, :, : n - L: 3] = math.nan
    other[:, :, 1: n - L: 3] = 1e30
    start = torch.rand(32, H, P, device=DEV, generator=g)

    def call(q, lse):
        return attention.attention_weights_paged(q, pool, table, lens, lse, start.clone(), k_scale=scale)
    want = call(q, blind)
    assert bool((want >= start).all()) and bool((want > start).any())
    assert torch.equal(call(q, lse), want) and torch.equal(call(other, lse), want)
