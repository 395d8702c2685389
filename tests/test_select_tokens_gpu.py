"""Selection of the tokens that stay (tq_select_tokens_cuda) against a stable sort."""
import math

import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _want(w, table, lens, keep, sinks, recent, width):
    P, H = w.shape[2], w.shape[1]
    out = torch.full((table.shape[0], H, width), -1, dtype=torch.int32)
    for b in range(table.shape[0]):
        L = lens[b]
        k = max(0, min(keep[b] if isinstance(keep, list) else keep, L, width))
        r = min(recent, k)
        s = min(sinks, k - r)
        some = k - r - s
        row = w[table[b].long()].transpose(0, 1).flatten(1)[:, :L].double().nan_to_num(-math.inf, math.inf, -math.inf)
        mid = row[:, s: L - r]
        order = torch.sort(mid, dim=1, descending=True, stable=True).indices[:, :some] + s
        for h in range(H):
            kept = torch.cat((torch.arange(s), order[h].sort().values.cpu(), torch.arange(L - r, L)))
            out[b, h, :k] = kept.to(torch.int32)
    return out


def _check(lens, H, P, keep, sinks=0, recent=0, width=None, seed=0, spread=2.0, fill=None, **kw):
    B = len(lens)
    per = max(1, -(-max(lens) // P))
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.exp(spread * torch.randn(B * per + 1, H, P, device=DEV, generator=g))
    if fill is not None:
        w = fill(w, g)
    table = torch.randperm(B * per + 1, generator=torch.Generator().manual_seed(seed))[: B * per].view(B, per).to(torch.int32).to(DEV)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    k = torch.tensor(keep, dtype=torch.int32, device=DEV) if isinstance(keep, list) else keep
    got = ops.select_tokens(w, table, kv_len, k, sinks=sinks, recent=recent, width=width, **kw)
    wide = width if isinstance(keep, list) or width is not None and width < keep else keep
    want = _want(w, table, lens, keep, sinks, recent, wide)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("lens", [[1], [16, 1, 0, 15], [513, 512, 511], [2049, 100, 4096], [5000, 8192, 8193]])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (5, 4, 0), (8, 4, 4), (100, 4, 32), (400, 0, 100), (6000, 3, 7)])
def test_matches_a_sort(lens, keep, sinks, recent):
    _check(lens, 2, 16, keep, sinks, recent, seed=keep)


@pytest.mark.parametrize("pairs,top", [((1, 8), 33000), ((3, 1), 100001), ((20, 8), 3001), ((1, 1), 70000)])
def test_clusters_of_all_sizes(pairs, top):
    _check([top] + [top // 2 + 1] * (pairs[0] - 1), pairs[1], 64, top // 5, 4, 128, seed=top)


def test_more_slots_than_a_cluster_holds():
    # over 8 x 40960 slots weights are read in every pass
    _check([340001, 5], 1, 1024, 50000, 4, 100, seed=1)


@pytest.mark.parametrize("kind", ["alike", "few", "zeros", "special", "steps"])
def test_ties_and_special_values(kind):
    def fill(w, g):
        u = torch.rand(w.shape, device=DEV, generator=g)
        if kind == "alike":
            return torch.ones_like(w)
        if kind == "few":
            return torch.where(u < 0.5, 0.25, torch.where(u < 0.9, 0.5, 0.75))
        if kind == "zeros":     # 0 and -0 are alike
            return torch.where(u < 0.4, 0.0, torch.where(u < 0.8, -0.0, w))
        if kind == "special":
            w = torch.where(u < 0.2, math.inf, torch.where(u < 0.4, -math.inf, w))
            return torch.where(u > 0.8, math.nan, torch.where(u > 0.7, -w, w))
        return (1.0 + torch.floor(u * 100) * 2.0 ** -23)     # neighbours among the floats
    for keep in (1, 200, 700, 1900):
        _check([2000, 777, 1900], 2, 32, keep, 2, 5, seed=3, fill=fill)


def test_numbers_to_keep_by_sequence():
    _check([500, 20, 300, 0], 2, 16, [100, 50, 0, 7], 4, 16, width=120, seed=1)
    _check([500, 20, 300, 9], 2, 16, [-5, 1000, 400, 3], 4, 16, width=350, seed=2)     # taken as the nearest of 0 .. width
    _check([500, 20], 2, 16, 100, 4, 16, width=60, seed=2)
    _check([500], 2, 16, 0, 4, 16, seed=2)
    # protected ones alone, and more of them than stay
    _check([500, 3], 2, 16, 10, 40, 40, seed=2)
    _check([500, 3], 2, 16, 50, 40, 20, seed=2)


def test_bounds_bad_pages_and_refusals():
    w = torch.rand(8, 2, 16, device=DEV)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    lens = torch.tensor([100], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    # lengths out of range are taken as the nearest
    over = ops.select_tokens(w, table, torch.tensor([1 << 30], dtype=torch.int32, device=DEV), 20, status=status)
    assert torch.equal(over, ops.select_tokens(w, table, torch.tensor([128], dtype=torch.int32, device=DEV), 20)) and int(status) == 0
    assert bool((ops.select_tokens(w, table, torch.tensor([-3], dtype=torch.int32, device=DEV), 20) == -1).all())
    # tokens behind the bound are left out
    short = ops.select_tokens(w, table, lens, 20, max_kv_len=64, status=status)
    assert int(status) == 1 and torch.equal(short, ops.select_tokens(w, table, torch.tensor([64], dtype=torch.int32, device=DEV), 20))
    # tokens of pages outside the pool go first
    bad = table.clone()
    bad[0, 2], bad[0, 4] = -1, 8
    status.zero_()
    got = ops.select_tokens(w, bad, lens, 68, status=status)
    want = [t for t in range(100) if t // 16 not in (2, 4)]
    assert int(status) == 1 and got[0].tolist() == [want, want]
    ops.select_tokens(w, bad, lens, 68)
    assert attention.last_status() == 1
    for change in (dict(weights=w.half()), dict(weights=w[:, :, ::2]), dict(page_table=table.long()), dict(kv_len=lens.long()), dict(keep=-1),
                   dict(keep=lens), dict(keep=lens.long(), width=4), dict(sinks=-1), dict(recent=-1), dict(max_kv_len=129),
                   dict(max_kv_len=-1), dict(out=torch.zeros(1, 2, 4, dtype=torch.int32, device=DEV)), dict(weights=w.cpu()),
                   dict(keep=lens, width=-1), dict(weights=torch.rand(8, 2, 24, device=DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.select_tokens(**{**dict(weights=w, page_table=table, kv_len=lens, keep=20), **change})
