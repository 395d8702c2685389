"""Attention over 8-bit pages, float32 and float16 outputs: queries enter the scores as two f16 terms.

Bound.  The second term leaves q' off by at most 2^-23 of its row's largest element, so what is left of float32 inputs'
error are the weights' roundings to f16: each evenly spread over +- half a step, at most 2^-11 of the weight, of variance
at most 2^-22 / 3 of its square.  They move an output by sum_j e_j p_j v_j, so the expected square of the whole error is
at most E = 2^-22 / 3 sum_j p_j^2 v_j^2 over all rows and elements.  The sums of squares below have 2048 outputs or more,
whose fluctuation about E is some 3 %; fp32 sums round to 2^-24 of terms that weights round to 2^-12 of, and scores of
size 10 to 2^-21.  Held to 1.25 sqrt(E).  (One f16 term alone moves scores of this size by 3 2^-12 of a query element's
share, three times as much as the bound.)
"""
import math

import pytest
import torch

from leankv_b200 import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [1, 5, 16, 150])   # 4 and 20 rows, 64 rows, 600 rows: the three kernels
def test_error_is_that_of_the_weights(n, D):
    B, H, grp, P, L = 2, 2, 4, 32, 2000
    g = torch.Generator(device=DEV).manual_seed(100 * D + n)
    per = -(-L // P)
    pool = lambda: (torch.randint(-127, 128, (B * per, H, P, D), dtype=torch.int8, device=DEV, generator=g),   # noqa: E731
                    torch.exp(0.3 * torch.randn(B * per, H, P // 16, device=DEV, generator=g)) / 75)
    (kp, ks), (vp, vs) = pool(), pool()
    table = torch.randperm(B * per, device=DEV, generator=g).to(torch.int32).view(B, per)
    q = 3 * torch.randn(B, H * grp, n, D, device=DEV, generator=g)
    lens = torch.full((B,), L, dtype=torch.int32, device=DEV)
    run = lambda x, dtype: attention.attention_q8_paged(x, kp, vp, ks, vs, table, lens, rotate_q=False, v_rotated=False,   # noqa: E731
                                                        out_dtype=dtype).double()
    got, half, rounded = run(q, torch.float32), run(q.half(), torch.float16), run(q.half(), torch.float32)
    err = most = 0.0
    for b in range(B):
        pg = table[b].long()
        k, v = ((c[pg].double() * s[pg].double().repeat_interleave(16, -1)[..., None]).transpose(0, 1).flatten(1, 2)[:, :L]
                for c, s in ((kp, ks), (vp, vs)))
        s = q[b].double().unflatten(0, (H, grp)) @ k[:, None].transpose(-1, -2) / math.sqrt(D)
        hide = torch.arange(L, device=DEV) > (L - n + torch.arange(n, device=DEV))[:, None]
        p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
        err += float((got[b].unflatten(0, (H, grp)) - p @ v[:, None]).square().sum())
        most += float((p.square() @ v.square()[:, None]).sum()) * 2.0 ** -22 / 3
    assert math.sqrt(err) <= 1.25 * math.sqrt(most)
    # the same kernel rounds its float32 answer once
    assert ((half - rounded).abs() <= 2.0 ** -11 * rounded.abs() + 2.0 ** -25).all()
