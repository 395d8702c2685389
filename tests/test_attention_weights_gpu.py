"""Sums of attention weights (tq_attention_weights_paged_cuda) against the formula in float64.

Tolerance.  A score's roundings: the Hadamard transform in fp32 (log2 D + 1 roundings of values of at most sum |q| / sqrt(D)), q'
divided by its largest element (two roundings of 2^-24) and taken as two f16 terms (what they leave is at most 2^-23 of the largest
element): (log2 D + 3) 2^-24 sum|q| / sqrt(D) + 2^-22 max|q'| on each element of q', times sum |k_d|.  TQ4 levels as two f16
terms are off by 2^-22 of each.  TQ2 and TQ3 levels are three terms of 8 bits, off by 2^-24 of the largest level, and products of
terms below 2^-23 of the largest level and element are left out; their sums are of whole numbers and exact, so that on these
inputs the part for the matrix instructions (D = 128: 25 times 2^-22 of the products' sizes) is far above both.  The products of a score are summed by at most 3 D / 16 matrix instructions, each off by at most
2^-22 of the sum of the products' sizes (8 bits: of codes + 128).  In the exponent four more roundings of 2^-24 of the sizes of
score and lse; the power 2^-22; the sum over the rows 2^-23 for each of them; the earlier weight's part 2^-23."""
import math

import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _hadamard(D):
    i = torch.arange(D, device=DEV)
    odd = torch.zeros(D, D, device=DEV, dtype=torch.int64)
    for bit in range(D.bit_length()):
        odd ^= ((i[:, None] & i) >> bit) & 1
    return (1 - 2 * odd).double() / math.sqrt(D)


def _keys(kind, pages, H, P, D, seed):
    """(pool, scale, values in float64, sizes that the products' sums are off by)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    if kind == 8:
        code = torch.randint(-127, 128, (pages, H, P, D), dtype=torch.int8, device=DEV, generator=g)
        scale = torch.exp(torch.randn(pages, H, P // 16, device=DEV, generator=g)) / 100
        wide = scale.double().repeat_interleave(16, -1)[..., None]
        return code, scale, code.double() * wide, (code.double().abs() + 128) * wide
    x = torch.randn(pages, H, P, D, device=DEV, generator=g) * 0.7
    pool = ops.quantize(x, kind)
    v = ops.dequantize(pool, kind).double()
    return pool, None, v, v.abs()


def _check(kind, B, H, grp, n, D, P, dtype, lens, q_len=None, fresh=None, decay=1.0, window=None, causal=True, rotate_q=True, sm=None,
           seed=0, lse_of=None, table=None, three=False, q_of=None):
    per = -(-max(16, max(lens)) // P)
    pool, scale, val, size = _keys(kind, B * per + 2, H, P, D, seed)
    g = torch.Generator().manual_seed(seed)
    if table is None:
        table = torch.randperm(B * per + 2, generator=g)[: B * per].view(B, per).to(torch.int32).to(DEV)
    gq = torch.Generator(device=DEV).manual_seed(seed + 2)
    q = torch.randn(B, n, H * grp, D, device=DEV, generator=gq).to(dtype).transpose(1, 2)
    if q_of is not None:
        q = q_of(q)
    w0 = torch.rand(B * per + 2, H, P, device=DEV, generator=gq)
    had, s_scale = _hadamard(D), D ** -0.5 if sm is None else sm
    want, tol = w0.double(), torch.zeros(w0.shape, device=DEV).double()
    lse = torch.full((B, H * grp, n), -math.inf, device=DEV)
    for b in range(B):
        L, m = lens[b], n if q_len is None else q_len[b]
        pg = table[b].long()
        k, sz = (t[pg].transpose(0, 1).flatten(1, 2)[:, :L] for t in (val, size))
        x = q[b].double() @ had if rotate_q else q[b].double()
        x = x.unflatten(0, (H, grp))
        s = s_scale * (x @ k[:, None].transpose(-1, -2))
        i = torch.arange(n, device=DEV)[:, None]
        sees = (torch.arange(L, device=DEV) <= (L - m + i if causal else L)) & (i < m)
        lse[b] = torch.logsumexp(s.masked_fill(~sees, -math.inf), -1).flatten(0, 1).float() if L else lse[b]
        if lse_of is not None:
            lse[b] = lse_of(lse[b])
        counts = sees & (i >= m - (window or n))
        l64 = lse[b].double().unflatten(0, (H, grp))[..., None]
        p = torch.where(counts & (l64 != -math.inf), torch.exp(s - l64), 0.0)
        q1 = q[b].double().abs().sum(-1).unflatten(0, (H, grp))[..., None] / math.sqrt(D)
        eq = (math.log2(D) + 3) * 2.0 ** -24 * q1 + 2.0 ** -22 * x.abs().amax(-1, keepdim=True)
        ds = abs(s_scale) * (eq * k.abs().sum(-1)[:, None, None]
                             + (3 * D / 16 + 1) * 2.0 ** -22 * (x.abs() @ sz[:, None].transpose(-1, -2)))
        ds = ds + 2.0 ** -22 * (s.abs() + l64.abs().nan_to_num(0.0, posinf=0.0))
        t = (p * (torch.expm1(ds) + 2.0 ** -22 + 2.0 ** -23 * grp * n)).sum((1, 2))
        slot = torch.arange(L, device=DEV)
        f = L if fresh is None else fresh[b]
        page = pg[slot // P]
        held = w0.double()[page, :, slot % P]
        kept = torch.where((slot < f)[:, None], held * decay, 0.0)
        got = p.sum((1, 2))
        want[page, :, slot % P] = kept + got.T
        tol[page, :, slot % P] = t.T + 2.0 ** -23 * (kept + got.T)
    w = w0.clone()
    args = dict(k_scale=scale, decay=decay, window=window, causal=causal, rotate_q=rotate_q, sm_scale=sm)
    if q_len is not None:
        args["q_len"] = torch.tensor(q_len, dtype=torch.int32, device=DEV)
    if fresh is not None:
        args["fresh"] = torch.tensor(fresh, dtype=torch.int32, device=DEV)
    out = attention.attention_weights_paged(q[:, :, 0] if three else q, pool, table, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                            lse[:, :, 0].contiguous() if three else lse, w, **args)
    assert out is w
    # slots behind the sequences, and pages of none, are as they were
    untouched = tol == 0
    assert torch.equal(w[untouched].double(), want[untouched])
    err = (w.double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), float((err - tol).max())
    return w


@pytest.mark.parametrize("kind", [8, 2, 3, 4])
@pytest.mark.parametrize("D,grp,P", [(128, 1, 16), (128, 4, 64), (256, 8, 16), (256, 3, 128), (128, 5, 32)])
def test_single_tokens(kind, D, grp, P):
    lens = [700, 1, 0, 129, 16]
    _check(kind, 5, 2, grp, 1, D, P, torch.bfloat16, lens, fresh=[699, 0, 0, 128, 15], decay=0.75, seed=grp, three=grp == 4)


@pytest.mark.parametrize("kind,D,grp,n", [(8, 128, 4, 5), (8, 128, 8, 9), (8, 256, 4, 33), (8, 128, 4, 130), (8, 256, 2, 300), (3, 128, 4, 20),
                                          (4, 256, 4, 20), (8, 128, 1, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows(kind, D, grp, n, causal):
    lens = [900, n, 20, 0, 301]
    _check(kind, 5, 2, grp, n, D, 32, torch.float16, lens, q_len=[n, n, n, n, 2 * n // 3], fresh=[900 - n, 0, 7, 0, 100], causal=causal, seed=n)


@pytest.mark.parametrize("kind", [2, 3, 4])
@pytest.mark.parametrize("D,grp,n,P", [(128, 3, 3, 16), (256, 8, 4, 64), (256, 5, 13, 16), (128, 16, 5, 128)])
def test_turboquant_rows(kind, D, grp, n, P):
    # one to three times the rows that are taken at a time; tokens of a CTA beyond the sums that it holds
    _check(kind, 3, 2, grp, n, D, P, torch.bfloat16, [4500, n, 17], q_len=[n, n, n - 1], fresh=[4500 - n, 0, 16], decay=0.5, seed=n)


@pytest.mark.parametrize("window", [1, 3, 40, 64, 99, 1000])
def test_window(window):
    n = 99
    _check(8, 4, 2, 4, n, 128, 64, torch.bfloat16, [3000, n, n + 500, 17], q_len=[n, n, 50, 0], window=window, decay=0.0, seed=window)


def test_long_sequences_and_many_rows_at_once():
    # tokens of a CTA beyond the sums that it holds at a time, rows beyond a chunk
    _check(8, 1, 1, 4, 40, 128, 64, torch.bfloat16, [9001], seed=1)
    _check(8, 40, 8, 4, 20, 128, 256, torch.bfloat16, [5000] * 40, seed=2)


@pytest.mark.parametrize("kind", [8, 3])
def test_scales_and_unrotated(kind):
    _check(kind, 2, 2, 4, 3 if kind == 8 else 1, 128, 16, torch.float32, [400, 33], rotate_q=False, sm=-0.05, seed=5)
    # scores of some size: weights from next to nothing to nearly one
    _check(kind, 2, 2, 4, 1, 128, 16, torch.float32, [400, 33], sm=1.5, seed=6)


def test_rows_that_saw_nothing_add_nothing():
    def some(lse):
        lse = lse.clone()
        lse[1] = -math.inf
        return lse
    _check(8, 2, 2, 4, 3, 128, 16, torch.bfloat16, [400, 33], lse_of=some, seed=7)


@pytest.mark.parametrize("kind,n", [(8, 1), (8, 5), (8, 70), (8, 300), (3, 1), (4, 9)])
def test_rows_that_saw_nothing_may_hold_anything(kind, n):
    B, H, P, D = 2, 2, 16, 128
    pool, scale, _, _ = _keys(kind, 20, H, P, D, 1)
    table = torch.arange(20, dtype=torch.int32, device=DEV).view(2, 10)
    g = torch.Generator(device=DEV).manual_seed(n)
    q = torch.randn(B, 4, n, D, device=DEV, generator=g)
    lens = torch.tensor([150, 140], dtype=torch.int32, device=DEV)
    lse = torch.rand(B, 4, n, device=DEV, generator=g) + 5.0
    lse[:, 1::2, : (n + 1) // 2] = -math.inf
    bad = q.clone()
    for i, x in enumerate((math.inf, -math.inf, math.nan)):
        bad[:, 1::2, i: (n + 1) // 2: 3, 7 * i] = x
    one, two = torch.rand(20, H, P, device=DEV, generator=g).repeat(2, 1, 1, 1)
    attention.attention_weights_paged(q, pool, table, lens, lse, one, k_scale=scale, causal=False)
    attention.attention_weights_paged(bad, pool, table, lens, lse, two, k_scale=scale, causal=False)
    assert bool(one.isfinite().all()) and torch.equal(one, two)


@pytest.mark.parametrize("kind,n", [(8, 5), (8, 16), (8, 100), (3, 5)])
def test_rows_of_unlike_sizes(kind, n):
    # each row keeps the accuracy of its own size
    def some(q):
        small = torch.arange(q.shape[1] * n, device=DEV).view(1, -1, n, 1) % 5 > 0
        return torch.where(small, q * 2.0 ** -10, q * 4)
    _check(kind, 2, 2, 4, n, 128, 32, torch.float32, [400, n], q_of=some, seed=n)


def test_earlier_weights_are_not_read_where_they_do_not_count():
    B, H, P, D = 1, 1, 16, 128
    pool, scale, _, _ = _keys(8, 4, H, P, D, 1)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(1, 4)
    q = torch.randn(B, 2, 1, D, device=DEV)
    lens = torch.tensor([50], dtype=torch.int32, device=DEV)
    w = torch.full((4, H, P), math.nan, device=DEV)
    lse = torch.zeros(B, 2, 1, device=DEV)
    attention.attention_weights_paged(q, pool, table, lens, lse, w, k_scale=scale, decay=0.0)
    assert bool(w.flatten()[:50].isfinite().all()) and bool(w.flatten()[50:].isnan().all())
    w.fill_(math.nan)
    attention.attention_weights_paged(q, pool, table, lens, lse, w, k_scale=scale, fresh=torch.zeros(1, dtype=torch.int32, device=DEV))
    assert bool(w.flatten()[:50].isfinite().all())


@pytest.mark.parametrize("kind,n", [(8, 1), (8, 70), (3, 1)])
def test_pages_outside_the_pool_hold_nothing(kind, n):
    B, H, P, D = 2, 2, 16, 128
    pool, scale, _, _ = _keys(kind, 20, H, P, D, 1)
    table = torch.arange(20, dtype=torch.int32, device=DEV).view(2, 10)
    bad = table.clone()
    bad[0, 3], bad[1, 0], bad[1, 9] = -1, 20, 1 << 30
    q = torch.randn(B, 4, n, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    lens = torch.tensor([150, 140], dtype=torch.int32, device=DEV)
    lse = torch.full((B, 4, n), 3.0, device=DEV)
    start = torch.rand(20, H, P, device=DEV)
    one, two = start.clone(), start.clone()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    attention.attention_weights_paged(q, pool, table, lens, lse, one, k_scale=scale, status=status)
    assert int(status) == 0
    attention.attention_weights_paged(q, pool, bad, lens, lse, two, k_scale=scale, status=status)
    assert int(status) == 1
    gone = torch.zeros(20, dtype=torch.bool, device=DEV)
    gone[3] = gone[10] = gone[19] = True
    assert torch.equal(two[gone], start[gone]) and torch.equal(two[~gone], one[~gone])
    assert attention.last_status() == 0
    attention.attention_weights_paged(q, pool, bad, lens, lse, two, k_scale=scale)
    assert attention.last_status() == 1 and attention.last_status() == 0


def test_refusals():
    pool, scale, _, _ = _keys(8, 4, 2, 16, 128, 1)
    q, lse = torch.zeros(1, 4, 3, 128, device=DEV), torch.zeros(1, 4, 3, device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(1, 4)
    lens, w = torch.tensor([20], dtype=torch.int32, device=DEV), torch.zeros(4, 2, 16, device=DEV)
    good = dict(q=q, k_pool=pool, page_table=table, kv_len=lens, lse=lse, weights=w, k_scale=scale)
    attention.attention_weights_paged(**good)
    for change in (dict(q=q[..., :64]), dict(q=q.double()), dict(q=q[:, :3].contiguous()), dict(k_pool=pool[:3]), dict(k_scale=None),
                   dict(k_scale=scale.half()), dict(lse=lse.half()), dict(lse=lse[:, :, :2]), dict(weights=w.half()), dict(weights=w[:, :1]),
                   dict(weights=w.transpose(0, 1)), dict(kv_len=lens.long()), dict(window=0), dict(window=-1), dict(decay=math.nan),
                   dict(sm_scale=math.inf), dict(max_kv_len=65), dict(page_table=table.long()), dict(q=q.cpu()), dict(weights=w.cpu()),
                   dict(k_pool=torch.zeros(4, 2, 16, 4, 14, dtype=torch.uint8, device=DEV)), dict(fresh=lens.long()),
                   dict(k_pool=torch.zeros(4, 2, 16, 4, 15, dtype=torch.uint8, device=DEV), k_scale=None)):
        with pytest.raises((ValueError, RuntimeError)):
            attention.attention_weights_paged(**{**good, **change})
