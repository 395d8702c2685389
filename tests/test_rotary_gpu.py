"""Rotary positions on the GPU (tq_rotary_cuda) against the formula in extended precision.

Tolerances count roundings.  cos and sin are rounded to float32 once (2^-24 relative), each product and the
sum once more: |error| <= 3 * 2^-24 * (|a| + |b|) for a pair (a, b), plus the rounding of the result to the
rows' type (eps / 2 of the value), plus the angle's own error p * 2^-64 turns.
"""
import math

import numpy as np
import pytest
import torch

from leankv_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _reference(x, positions, freq, axis, interleaved, inverse, scale=1.0):
    """Rotated rows in float64 from angles in extended precision; also |a| + |b| of each element's pair."""
    pos = positions.cpu().numpy().astype(np.longdouble)
    f = freq.cpu().numpy().astype(np.longdouble)
    if pos.ndim == 2:
        pos = pos[None]
    ax = np.zeros(len(f), dtype=int) if axis is None else axis.cpu().numpy()
    angle = np.stack([pos[ax[i]] * f[i] for i in range(len(f))], -1)   # [B, n, pairs]
    if inverse:
        angle = -angle
    cos = torch.from_numpy(np.cos(angle).astype(np.float64))[:, None] * scale
    sin = torch.from_numpy(np.sin(angle).astype(np.float64))[:, None] * scale
    y = x.cpu().double()
    R = 2 * len(f)
    lo = slice(0, R, 2) if interleaved else slice(0, R // 2)
    hi = slice(1, R, 2) if interleaved else slice(R // 2, R)
    a, b = y[..., lo].clone(), y[..., hi].clone()
    out, size = y.clone(), torch.zeros_like(y)
    out[..., lo], out[..., hi] = a * cos - b * sin, b * cos + a * sin
    size[..., lo] = size[..., hi] = (a.abs() + b.abs()) * abs(scale)
    return out, size


def _check(got, x, positions, freq, axis=None, interleaved=False, inverse=False, scale=1.0):
    want, size = _reference(x, positions, freq, axis, interleaved, inverse, scale)
    far = float(positions.abs().max()) * 2.0 ** -64 * 2 * math.pi
    half = torch.finfo(got.dtype).eps / 2
    err = (got.cpu().double() - want).abs()
    # the last factor: a subnormal result of the type is off by half its smallest step
    tol = (3 * 2.0 ** -24 + far) * size + half * want.abs() * (1 + 2.0 ** -10) + torch.finfo(got.dtype).smallest_normal * half * 2
    # elements that do not turn are copied
    R = 2 * freq.numel()
    assert torch.equal(got[..., R:].cpu(), x[..., R:].cpu())
    bad = err > tol + half * size * 4 * 2.0 ** -24
    assert not bool(bad.any()), (err / tol).max()


def _inputs(B, H, n, D, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(B, H, n, D, device=DEV, generator=g).mul(3).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,R,interleaved", [(128, 128, False), (128, 64, True), (256, 256, True), (64, 16, False),
                                             (80, 80, False), (72, 48, True), (512, 512, False), (256, 48, False)])
@pytest.mark.parametrize("n", [1, 17, 70])
def test_rotary_matches_formula(dtype, D, R, interleaved, n):
    B, H = 2, 3
    x = _inputs(B, H, n, D, dtype, D + R + n)
    freq = ops.rotary_frequencies(R, device=DEV)
    pos = torch.randint(0, 5000, (B, n), device=DEV, dtype=torch.int32, generator=torch.Generator(device=DEV).manual_seed(n))
    rope = ops.Rotary(freq, interleaved=interleaved)
    _check(ops.rotary(x, pos, rope), x, pos, freq, interleaved=interleaved)
    _check(ops.rotary(x, pos, rope, inverse=True), x, pos, freq, interleaved=interleaved, inverse=True)


def test_rotary_axes_and_scale():
    B, H, n, D = 2, 4, 45, 128
    x = _inputs(B, H, n, D, torch.bfloat16, 1)
    freq = ops.rotary_frequencies(D, theta=500000.0, device=DEV)
    pos = torch.randint(-300, 3000, (3, B, n), device=DEV, dtype=torch.int32)
    for mixed in (False, True):
        axis = ops.rotary_axes((16, 24, 24), DEV, mixed)
        rope = ops.Rotary(freq, axis, scale=1.25)
        _check(ops.rotary(x, pos, rope), x, pos, freq, axis, scale=1.25)


@pytest.mark.parametrize("first", [2 ** 20, 2 ** 27, 2 ** 31 - 40, -2 ** 31])
def test_rotary_far_positions(first):
    """Angles are those of the integer position: nothing is lost to its size."""
    x = _inputs(1, 2, 33, 128, torch.float32, 3)
    freq = torch.cat([ops.rotary_frequencies(96, device=DEV), torch.tensor([1e-9, 3.7, 100.0, 0.0], device=DEV).double(),
                      torch.rand(12, device=DEV).double()])
    pos = (torch.arange(33, device=DEV, dtype=torch.int64) + first).to(torch.int32).view(1, 33)
    _check(ops.rotary(x, pos, ops.Rotary(freq)), x, pos, freq)


def test_rotary_views_in_place_and_both_tensors():
    """Queries and keys as views of one projection's output, rotated in place; the values stay."""
    B, n, hq, hk, D = 3, 21, 8, 2, 128
    qkv = _inputs(B, n, hq + 2 * hk, D, torch.bfloat16, 5)
    before = qkv.clone()
    q, k, _ = (t.transpose(1, 2) for t in qkv.split([hq, hk, hk], dim=2))
    freq = ops.rotary_frequencies(D, device=DEV)
    pos = torch.randint(0, 900, (B, n), device=DEV, dtype=torch.int32)
    a, b = ops.rotary(q.contiguous(), pos, ops.Rotary(freq), k=k.contiguous())
    r, s = ops.rotary(q, pos, ops.Rotary(freq), k=k, out=q, k_out=k)
    assert r.data_ptr() == q.data_ptr() and torch.equal(q, a) and torch.equal(k, b)
    _check(a, before[:, :, :hq].transpose(1, 2), pos, freq)
    _check(b, before[:, :, hq:hq + hk].transpose(1, 2), pos, freq)
    assert torch.equal(qkv[:, :, hq + hk:], before[:, :, hq + hk:])


@pytest.mark.parametrize("interleaved,scale", [(False, 1.0), (True, 0.75)])
def test_rotary_inverse_is_the_gradient(interleaved, scale):
    """The rotation is linear: its gradient against autograd of the formula, and against differences."""
    B, H, n, D = 2, 2, 9, 128
    x = _inputs(B, H, n, D, torch.float32, 7)
    w = _inputs(B, H, n, D, torch.float32, 8)
    freq = ops.rotary_frequencies(64, device=DEV)
    pos = torch.randint(0, 40000, (B, n), device=DEV, dtype=torch.int32)
    rope = ops.Rotary(freq, interleaved=interleaved, scale=scale)
    grad = ops.rotary(w, pos, rope, inverse=True)
    z = x.cpu().double().requires_grad_()
    angle = pos.cpu().double()[..., None] * freq.cpu()
    c, s = angle.cos()[:, None] * scale, angle.sin()[:, None] * scale
    lo, hi = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    y = torch.cat([z[..., lo] * c - z[..., hi] * s, z[..., hi] * c + z[..., lo] * s, z[..., 64:]], -1)
    wl = torch.cat([w[..., lo], w[..., hi], w[..., 64:]], -1).cpu().double()
    (y * wl).sum().backward()
    # 64-bit angles of positions below 2^16 are off by at most 2^16 * 2^-53
    tol = 4 * 2.0 ** -24 * 2 * w.abs().max().item()
    assert (grad.cpu().double() - z.grad).abs().max().item() <= tol
    # a step along one element changes sum(w * rotary(x)) by its gradient (linear, so the step may be large);
    # 1/8 is exact, each of the two sums of 64 * 36 float32 terms is taken in 64 bits
    for at in [(0, 0, 3, 1), (1, 1, 8, 33), (0, 1, 0, 63), (1, 0, 5, 100)]:
        up, down = x.clone(), x.clone()
        up[at] = x[at] + 8
        down[at] = x[at] - 8
        f = [(ops.rotary(t, pos, rope).double() * w.double()).sum().item() for t in (up, down)]
        step = (up[at].double() - down[at].double()).item()
        # two results change, each rounded three times at magnitudes up to 8 + |x|
        lim = 2 * 2 * 3 * 2.0 ** -24 * (8 + 2 * x.abs().max().item()) * w.abs().max().item() / step
        assert abs((f[0] - f[1]) / step - grad[at].item()) <= lim + tol


def test_rotary_graph_replay_and_stream():
    x = _inputs(2, 4, 8, 128, torch.float16, 11)
    freq = ops.rotary_frequencies(128, device=DEV)
    pos = torch.zeros(2, 8, dtype=torch.int32, device=DEV)
    rope, out = ops.Rotary(freq), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rotary(x, pos, rope, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary(x, pos, rope, out=out)
    for first in (0, 77, 123456):
        pos.copy_(torch.arange(8, device=DEV, dtype=torch.int32) + first)
        graph.replay()
        assert torch.equal(out, ops.rotary(x, pos, rope))


def test_rotary_empty_and_refusals():
    freq = ops.rotary_frequencies(64, device=DEV)
    rope = ops.Rotary(freq)
    x = _inputs(2, 2, 4, 64, torch.float16, 1)
    pos = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    assert ops.rotary(x[:, :, :0], pos[:, :0].contiguous(), rope).shape == (2, 2, 0, 64)
    assert ops.rotary(x[:0], pos[:0], rope).shape == (0, 2, 4, 64)
    bad = [dict(q=x.double()), dict(q=x[0]), dict(q=x.transpose(2, 3)), dict(positions=pos.long()),
           dict(positions=pos[:1]), dict(positions=pos.expand(3, 2, 4).contiguous()), dict(positions=None),
           dict(rope=ops.Rotary(freq.float())), dict(rope=ops.Rotary(freq, axis=freq)), dict(k=x[:, :, :2]),
           dict(k=x.float()), dict(out=x.float()), dict(out=x[:1].expand(2, 2, 4, 64)), dict(q=x.cpu()), dict(rope=ops.Rotary(freq.cpu()))]
    for change in bad:
        with pytest.raises(ValueError):
            ops.rotary(**{**dict(q=x, positions=pos, rope=rope), **change})
    wide = torch.zeros(2, 2, 4, 68, dtype=torch.float16, device=DEV)
    for change in (dict(q=wide[..., 1:65]), dict(q=wide[..., :64]), dict(rope=ops.Rotary(freq[:20].contiguous())),
                   dict(rope=ops.Rotary(ops.rotary_frequencies(128, device=DEV))),
                   dict(out=x, q=x[:, :, :4].transpose(0, 1).contiguous().transpose(0, 1), positions=pos)):
        if "out" in change:
            continue
        with pytest.raises(ops.L.TQError):
            ops.rotary(**{**dict(q=x, positions=pos, rope=rope), **change})
    with pytest.raises(ops.L.TQError):   # in place at other strides
        y = torch.zeros(2, 4, 4, 64, dtype=torch.float16, device=DEV)
        ops.rotary(y[:, ::2, :, :], pos, rope, out=y[:, :2])
