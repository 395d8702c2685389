"""Rows of one token, one head or one sequence in views whose stride in that dimension is odd: no step is ever taken along
it, so the calls go through and give what they give for packed copies."""
import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def _view(B, H, n, seed, dtype=torch.bfloat16):
    """[B, H, n, D] whose strides of dimensions of one are odd."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(B, H, n, D, device=DEV, generator=g).to(dtype)
    odd = [s if k > 1 else 3 * D + 1 + i for i, (k, s) in enumerate(zip((B, H, n), x.stride()))]
    y = x.as_strided((B, H, n, D), (*odd, 1))
    assert torch.equal(x, y)
    return y


SHAPES = [(1, 4, 3), (3, 1, 5), (2, 4, 1), (1, 1, 1), (1, 1, 40)]


@pytest.mark.parametrize("B,H,n", SHAPES)
def test_rotary(B, H, n):
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    pos = torch.arange(B * n, dtype=torch.int32, device=DEV).view(B, n)
    q, k = _view(B, H, n, 1), _view(B, 1, n, 2)
    want = ops.rotary(q.contiguous().clone(), pos, rope, k=k.contiguous().clone())
    got = ops.rotary(q, pos, rope, k=k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = _view(B, H, n, 3)
    assert torch.equal(ops.rotary(q, pos, rope, out=out), want[0])
    # in place, through another view of the same rows
    assert torch.equal(ops.rotary(q, pos, rope, out=q.as_strided(q.shape, [s if m > 1 else 64 for m, s in zip(q.shape, q.stride())])),
                       want[0]) and torch.equal(q, want[0])


@pytest.mark.parametrize("kt", [3, 8])
@pytest.mark.parametrize("B,H,n", SHAPES)
def test_append(B, H, n, kt):
    P, per = 16, 4
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    table = torch.arange(B * per, dtype=torch.int32, device=DEV).view(B, per)
    pos = torch.full((B,), 5, dtype=torch.int32, device=DEV)
    q, k, v = _view(B, 4 * H, n, 1), _view(B, H, n, 2), _view(B, H, n, 3)
    got = []
    for rows in ((q, k, v), tuple(t.contiguous().clone() for t in (q, k, v))):
        if kt == 8:
            pools = [torch.zeros(B * per, H, P, D, dtype=torch.int8, device=DEV) for _ in range(2)]
            scales = dict(k_scale=torch.zeros(B * per, H, 1, device=DEV), v_scale=torch.zeros(B * per, H, 1, device=DEV))
        else:
            pools = [torch.zeros(B * per, H, P, D // 32, b, dtype=torch.uint8, device=DEV) for b in (14, 18)]
            scales = {}
        out = ops.kv_append_rotary_paged(rows[1], rows[2], *pools, table, pos, rope=rope, q=rows[0], **scales)
        got.append([out, *pools, *scales.values()])
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert got[0][1].any() and got[0][2].any()


@pytest.mark.parametrize("B,H,n", SHAPES)
def test_attention(B, H, n):
    P, per = 16, 4
    g = torch.Generator(device=DEV).manual_seed(4)
    kp, vp = (torch.randint(-127, 128, (B * per, H, P, D), dtype=torch.int8, device=DEV, generator=g) for _ in range(2))
    ks, vs = (torch.rand(B * per, H, 1, device=DEV, generator=g) / 100 for _ in range(2))
    table = torch.arange(B * per, dtype=torch.int32, device=DEV).view(B, per)
    lens = torch.full((B,), 50, dtype=torch.int32, device=DEV)
    q = _view(B, H, n, 1)
    want = attention.attention_q8_paged(q.contiguous().clone(), kp, vp, ks, vs, table, lens)
    out = _view(B, H, n, 5)
    assert torch.equal(attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens), want)
    assert torch.equal(attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, out=out), want)


def test_odd_strides_that_are_used_are_refused():
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    x = torch.zeros(2, 1, 2 * (D + 1), dtype=torch.bfloat16, device=DEV).as_strided((2, 1, 2, D), (2 * D + 2, D, D + 1, 1))
    with pytest.raises(ops.L.TQError):
        ops.rotary(x, torch.zeros(2, 2, dtype=torch.int32, device=DEV), rope)
