"""Heads whose values are all zero (scales of 0) behind long caches whose scores rise after the first tokens: the sum of
the weights stays within float32, whatever stands in for the scale.

A row's running maximum follows scores only when they exceed it by more than 8 (base 2), so weights of up to 2^14 are
summed over all tokens.  The answer is 0 and the log-sum-exp log(128 + (L - 128) 2^7.9), off by the scores' roundings (one
code of 127 and a power-of-two query: below 2^-20 of 7.9) and fp32 sums (2^-14, as in the other tests).
"""
import math

import pytest
import torch

from leankv_b200 import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [128, 256])
# sequences that share one cache (so that its tokens are split over few CTAs or none), query tokens: each kernel
@pytest.mark.parametrize("B,n", [(600, 1), (100, 1), (150, 16), (40, 120)])
def test_long_cache_of_zero_values(B, n, D):
    L, P, grp = 131072, 512, 4
    kp = torch.zeros(L // P, 1, P, D, dtype=torch.int8, device=DEV)
    kp[:, :, :, 0] = 127
    kp[0, :, :128, 0] = 0   # every warp's first block, a tile
    ks = torch.full((L // P, 1, P // 16), 7.9 * math.log(2.0) / 127, device=DEV)
    vp, vs = torch.zeros_like(kp), torch.zeros_like(ks)
    table = torch.arange(L // P, dtype=torch.int32, device=DEV).expand(B, -1).contiguous()
    lens = torch.full((B,), L, dtype=torch.int32, device=DEV)
    q = torch.zeros(B, grp, n, D, device=DEV)
    q[..., 0] = 1.0
    out, lse = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, causal=False, rotate_q=False, sm_scale=1.0,
                                            return_lse=True)
    assert bool((out == 0).all())
    want = math.log(128 + (L - 128) * 2.0 ** 7.9)
    assert float((lse.double() - want).abs().max()) <= 2.0 ** -14 + 7.9 * 2.0 ** -20
    # a head with values beside them: one block in the middle
    vp[40], vs[40, :, :1] = 100, 0.01
    vp[40, :, 16:] = 0
    out, lse = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, causal=False, rotate_q=False, v_rotated=False,
                                            sm_scale=1.0, return_lse=True)
    share = 16 * 2.0 ** 7.9 / (128 + (L - 128) * 2.0 ** 7.9)
    # weights and their sum: f16 and the tolerances above
    assert float((out.double() / share - 1).abs().max()) <= 2.0 ** -11 + 2.0 ** -13
    assert float((lse.double() - want).abs().max()) <= 2.0 ** -14 + 7.9 * 2.0 ** -20
