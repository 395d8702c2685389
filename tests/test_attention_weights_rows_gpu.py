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


@pytest.mark.parametrize("D", [128, 256])
def test_scores_are_rounded_to_the_nearest(D):
    """Scores' last places of many rows, where q' is exact in its three 8-bit terms: elements are whole multiples of 2^-14 with a largest
    one of 127, rows are not rotated, and codes are small, so that the products' sums are below 2^10.  In units of 2^-7 of the first
    term's, a score is then off by at most half for the joining of the terms, and by fp32's roundings: of the sum (2^-15 of the first
    term's unit: 2^-8), of the factor and its product with a scale and the sum (four of 2^-24 of up to 2^10: 2^-5), of the power's argument
    (below 2^3, in scores of 2^-8 a unit: 2^-8), of the power (2^-22 / 2^-15: 2^-7) and of at most 12 sums over rows (12 * 2^-24 / 2^-15: 0.024):
    together below 1/8.  Errors are spread over both sides: of T tokens their mean is off by at most about 6 / sqrt(12 T)."""
    P, L, grp, n = 128, 4096, 8, 16
    g = torch.Generator(device=DEV).manual_seed(D)
    code = torch.randint(-1, 2, (L // P, 1, P, D), dtype=torch.int8, device=DEV, generator=g)
    unit = 2.0 ** -8                      # of the products' sums, in scores
    scale = torch.ones(L // P, 1, P // 16, device=DEV)
    row = torch.randint(-(24 << 14), (24 << 14) + 1, (D,), device=DEV, generator=g).double() / 2 ** 14
    row[5] = 127.0
    q = row.float().expand(1, grp, n, D).contiguous()
    assert torch.equal(q[0, 0, 0].double(), row)
    table = torch.arange(L // P, dtype=torch.int32, device=DEV).view(1, -1)
    s = code.double().flatten(0, 2) @ row * unit
    assert float((s / unit).abs().max()) < 2 ** 10
    w = torch.zeros(L // P, 1, P, device=DEV)
    attention.attention_weights_paged(q, code, table, torch.tensor([L], dtype=torch.int32, device=DEV), torch.zeros(1, grp, n, device=DEV), w,
                                      k_scale=scale, causal=False, rotate_q=False, sm_scale=unit)
    # all rows alike: a token's weight is their number times one power
    err = (torch.log(w.double().flatten() / (grp * n)) - s) / (unit * 2.0 ** -7)
    assert float(err.abs().max()) <= 0.5 + 1 / 8
    assert abs(float(err.mean())) <= 6 / math.sqrt(12 * L)
