"""Masks and depths of drafted trees (tq_draft_tree_cuda) against walking up the parents, and attention of trees over 8-bit
pages (tq_attention_q8_tree_paged_cuda) against the formula in float64.

Tolerance of the attention, as derived in test_attention_q8_gpu.py: scores off by at most ds = sm_scale * 2^-12 max|q'| * sum |k_d|, so
weights by e^(2 ds) and the roundings to f16 (2^-11) and of the fp32 sums (2^-14), all of sum_j p_j |v_j|; weights below f16's
normal numbers by 2^-31 max_j(p_j vs_j) sum_j |code_j|; half a step of the output type."""
import math

import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _parents(B, n, seed, width=6):
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(n)
    p = torch.maximum(i - 1 - torch.randint(0, width, (B, n), generator=g), torch.tensor(-1))
    p[torch.rand(B, n, generator=g) < 0.1] = -1
    return p.to(torch.int32)


def _ancestors(parents):
    B, n = parents.shape
    seen = torch.zeros(B, n, n, dtype=torch.bool)
    for b in range(B):
        for i in range(n):
            p = int(parents[b, i])
            if 0 <= p < i:
                seen[b, i] = seen[b, p]
            seen[b, i, i] = True
    return seen


def _bits(mask, n):
    return ((mask.cpu()[..., None] >> torch.arange(32, dtype=torch.int32)) & 1).flatten(-2)[..., :n].bool()


@pytest.mark.parametrize("B,n", [(1, 1), (3, 2), (2, 31), (2, 32), (5, 33), (1, 128), (2, 129), (1, 700)])
def test_masks_and_depths(B, n):
    parents = _parents(B, n, n)
    if n > 2:
        parents[0, 1], parents[0, 2] = 5000, 2     # neither comes before its node: roots
    got = ops.draft_tree(parents.to(DEV))
    want = _ancestors(parents)
    assert got.mask.shape == (B, n, -(-n // 32)) and torch.equal(_bits(got.mask, n), want)
    assert torch.equal(got.depth.cpu(), want.sum(-1).to(torch.int32) - 1)


def test_chain_of_the_longest_and_one_tree_for_all():
    n = 4096
    got = ops.draft_tree(torch.arange(-1, n - 1, dtype=torch.int32, device=DEV))
    assert torch.equal(got.depth.cpu(), torch.arange(n, dtype=torch.int32)[None])
    assert torch.equal(_bits(got.mask, n), torch.ones(n, n, dtype=torch.bool).tril()[None])
    # a view with rows further apart
    wide = _parents(3, 40, 1).to(DEV).repeat(1, 2)
    assert torch.equal(ops.draft_tree(wide[:, :40]).mask, ops.draft_tree(wide[:, :40].contiguous()).mask)
    assert ops.draft_tree(torch.zeros(0, 5, dtype=torch.int32, device=DEV)).mask.shape == (0, 5, 1)
    for bad in (torch.zeros(1, 4097, dtype=torch.int32, device=DEV), torch.zeros(2, 3, device=DEV),
                torch.zeros(2, 6, dtype=torch.int32, device=DEV)[:, ::2]):
        with pytest.raises((ValueError, RuntimeError)):
            ops.draft_tree(bad)


def _hadamard(D):
    i = torch.arange(D, device=DEV)
    odd = torch.zeros(D, D, device=DEV, dtype=torch.int64)
    for bit in range(D.bit_length()):
        odd ^= ((i[:, None] & i) >> bit) & 1
    return (1 - 2 * odd).double() / math.sqrt(D)


def _pools(pages, H, P, D, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    code = torch.randint(-127, 128, (pages, H, P, D), dtype=torch.int8, device=DEV, generator=g)
    return code, torch.exp(torch.randn(pages, H, P // 16, device=DEV, generator=g)) / 100


def _check(B, H, grp, n, D, P, dtype, lens, q_len, seen, mask, seed=0, pages_off=0):
    top = max(16, max(lens))
    per = -(-top // P)
    kp, ks = _pools(B * per + 1, H, P, D, seed)
    vp, vs = _pools(B * per + 1, H, P, D, seed + 1)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * per + 1, generator=g)[: B * per].view(B, per).to(torch.int32).to(DEV)
    gq = torch.Generator(device=DEV).manual_seed(seed + 2)
    q = torch.randn(B, n, H * grp, D, device=DEV, generator=gq).to(dtype).transpose(1, 2)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ql = None if q_len is None else torch.tensor(q_len, dtype=torch.int32, device=DEV)
    got, lse = attention.attention_q8_paged(q, kp, vp, ks, vs, table, kv_len, q_len=ql, return_lse=True, tree=mask)
    had = _hadamard(D)
    half = torch.finfo(dtype).eps / 2
    for b in range(B):
        L, m = lens[b], n if q_len is None else q_len[b]
        base = L - m
        # (tokens before the cache's first are none; neither are the nodes that would lie there)
        sees = torch.zeros(n, L, dtype=torch.bool)
        for i in range(m):
            if base + i >= 0:
                sees[i, :max(base, 0)] = True
                lo = max(0, -base)
                sees[i, base + lo:] = seen[b if len(seen) > 1 else 0, i, lo:m]
        sees = sees.to(DEV)
        pg = table[b].long()
        k, v = ((c[pg].double() * s[pg].double().repeat_interleave(16, -1)[..., None]).transpose(0, 1).flatten(1, 2)[:, :L]
                for c, s in ((kp, ks), (vp, vs)))
        x = (q[b].double() @ had).unflatten(0, (H, grp))
        s = (D ** -0.5 * (x @ k[:, None].transpose(-1, -2))).masked_fill(~sees, -math.inf)
        ds = D ** -0.5 * 2.0 ** -12 * x.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None, None]
        e = ds.masked_fill(~sees, 0.0).amax(-1, keepdim=True) if L else torch.zeros(H, grp, n, 1, device=DEV).double()
        p = torch.softmax(s, -1).nan_to_num(0.0)
        o, tol = p @ v[:, None], (torch.expm1(2 * e) + 2.0 ** -11 + 2.0 ** -14) * (p @ v.abs()[:, None])
        if L:
            step = vs[pg].double().repeat_interleave(16, -1).transpose(0, 1).flatten(1, 2)[:, :L]
            codes = vp[pg].double().transpose(0, 1).flatten(1, 2)[:, :L].abs().sum(1)
            tol = tol + 2.0 ** -31 * (p * step[:, None, None]).amax(-1, keepdim=True) * codes[:, None, None]
        o, tol = (o @ had).flatten(0, 1), (tol @ had.abs()).flatten(0, 1)
        err = (got[b].double() - o).abs()
        assert bool((err <= tol * (1 + half) + half * o.abs() + 1e-30).all()), (b, float((err - tol).max()))
        want = torch.logsumexp(s, -1).flatten(0, 1) if L else torch.full((H * grp, n), -math.inf, device=DEV).double()
        empty = want == -math.inf
        assert torch.equal(lse[b] == -math.inf, empty) and bool((got[b][empty] == 0).all())
        assert bool(((lse[b].double() - want).abs()[~empty] <= (e.squeeze(-1).flatten(0, 1) + 2.0 ** -14)[~empty]).all())


# few rows, rows converted by the kernel, and tiles; a group that does not divide the tiles
@pytest.mark.parametrize("D,grp,n", [(128, 1, 1), (128, 4, 7), (128, 4, 12), (128, 1, 48), (256, 2, 16), (256, 1, 32), (128, 3, 17), (128, 4, 33),
                                     (256, 4, 13), (128, 1, 128), (128, 8, 60), (256, 8, 64), (128, 5, 200)])
@pytest.mark.parametrize("P,dtype", [(16, torch.bfloat16), (64, torch.float16)])
def test_trees_of_all_sizes(D, grp, n, P, dtype):
    # a long prefix, one that ends inside a block, none, nodes without a place in the cache, padding
    lens = [600 + n, 37 + n, n, max(1, n - 3), 300 + (n + 1) // 2]
    q_len = [n, n, n, n, (n + 1) // 2]
    parents = _parents(5, n, D + n)
    _check(5, 2, grp, n, D, P, dtype, lens, q_len, _ancestors(parents), ops.draft_tree(parents.to(DEV)), seed=n)


@pytest.mark.parametrize("grp,n", [(4, 9), (4, 40), (8, 90)])
def test_masks_of_ones_own(grp, n):
    """Any bits: rows that see nothing but the prefix, later nodes, nodes behind the sequence's count (ignored)."""
    g = torch.Generator().manual_seed(n)
    seen = torch.rand(1, n, n, generator=g) < 0.4
    seen[0, 3] = False
    words = torch.nn.functional.pad(seen, (0, -n % 32)).unflatten(-1, (-1, 32)).long() << torch.arange(32)
    mask = words.sum(-1).to(torch.int32).to(DEV)
    # the second sequence has no prefix: its row 3 sees nothing; the third has no row at all
    _check(3, 2, grp, n, 128, 16, torch.bfloat16, [200 + n, n, 0], [n, n - 1, 0], seen, mask, seed=n + 1)


@pytest.mark.parametrize("grp,n", [(4, 5), (4, 30), (8, 70)])
def test_a_chain_is_the_causal_call(grp, n):
    B, H, D, P = 2, 2, 128, 32
    kp, ks = _pools(40, H, P, D, 1)
    vp, vs = _pools(40, H, P, D, 2)
    table = torch.arange(40, dtype=torch.int32, device=DEV).view(2, 20)
    lens = torch.tensor([500, n + 1], dtype=torch.int32, device=DEV)
    q = torch.randn(B, H * grp, n, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).bfloat16()
    tree = ops.draft_tree(torch.arange(-1, n - 1, dtype=torch.int32, device=DEV))
    a = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens)
    b = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, tree=tree)
    # the same products; where a split's end depends on the row tile's last token sums may be taken in another order
    assert float((a.float() - b.float()).norm() / a.float().norm()) < 2.0 ** -8


def test_refusals():
    kp, ks = _pools(4, 1, 16, 128, 0)
    q = torch.zeros(2, 2, 5, 128, device=DEV, dtype=torch.bfloat16)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    lens = torch.tensor([9, 9], dtype=torch.int32, device=DEV)
    call = lambda tree, **kw: attention.attention_q8_paged(q, kp, kp, ks, ks, table, lens, tree=tree, **kw)   # noqa: E731
    good = torch.zeros(2, 5, 1, dtype=torch.int32, device=DEV)
    call(good)
    for bad in (good.long(), good[:, :4], good.expand(2, 5, 2), torch.zeros(3, 5, 1, dtype=torch.int32, device=DEV), good[0],
                torch.zeros(2, 5, 2, dtype=torch.int32, device=DEV)[..., :1]):
        with pytest.raises(ValueError):
            call(bad)
    with pytest.raises(ValueError):
        call(good.cpu())
    with pytest.raises(ValueError):
        call(good, causal=False)
