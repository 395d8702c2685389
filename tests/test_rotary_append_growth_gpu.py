"""8-bit pages whose block scales grow at every step, in many units at once: every lane of a unit has to take the scale
that the block had before the step, whenever it comes to read it.

The codes and scales of each step equal, one by one, a plain restatement that starts from the step's own rows: scale
max(old, max |x| / 127), new codes round(x / scale), older codes round(code * (old / scale)) in float32 operations.
"""
import pytest
import torch

from leankv_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [1, 3])
def test_older_codes_follow_every_growth(D, n):
    B, H, P = 96, 8, 16
    table = torch.randperm(B, generator=torch.Generator().manual_seed(D)).to(torch.int32).view(B, 1).to(DEV)
    kp, vp = (torch.zeros(B, H, P, D, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(B, H, 1, device=DEV) for _ in range(2))
    want = [(t[table[:, 0].long()].clone(), s[table[:, 0].long(), :, 0].clone()) for t, s in ((kp, ks), (vp, vs))]
    gen = torch.Generator(device=DEV).manual_seed(7 * D + n)
    for first in range(0, P - n + 1, n):
        pos = torch.full((B,), first, dtype=torch.int32, device=DEV)
        # rows of float32 values that no transform changes: rotate=False; each step is larger than the one before
        rows = [torch.randn(B, H, n, D, device=DEV, generator=gen) * (1.0 + 0.37 * first) for _ in range(2)]
        ops.kv_append_rotary_paged(rows[0], rows[1], kp, vp, table, pos, k_scale=ks, v_scale=vs, rotate=False)
        for i, x in enumerate(rows):
            code, old = want[i]
            new = torch.maximum(old, x.abs().amax((-1, -2)) * torch.tensor(1.0 / 127.0, device=DEV))
            inv = 1.0 / new
            code[:, :, :first] = torch.round(code[:, :, :first].float() * (old * inv)[..., None, None]).to(torch.int8)
            code[:, :, first:first + n] = torch.round(x * inv[..., None, None]).clamp(-127, 127).to(torch.int8)
            want[i] = (code, new)
            pool, scale = (kp, ks) if i == 0 else (vp, vs)
            assert torch.equal(scale[table[:, 0].long(), :, 0], new)
            assert torch.equal(pool[table[:, 0].long()], code), (first, i)
