"""Prompts over 8-bit pages where there are rows enough for two row tiles a CTA (heads of 128, bfloat16 outputs; half as
many CTAs of 256 rows as the GPU has SMs), against the formula with the tolerances of test_attention_q8_gpu."""
import pytest
import torch
from test_attention_q8_gpu import _check, _pools, _q, _reference, _table

from leankv_b200 import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def _two_tiles(pairs, rows):
    return rows >= 449 and 2 * pairs * -(-rows // 256) >= torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("grp,n,top", [(4, 257, 700), (1, 1100, 1100), (8, 140, 2000), (3, 350, 352)])
def test_prompts_match_formula(grp, n, top, P):
    """Second row tiles of a few rows or of none, prefixes, lengths that end inside tiles, sequences shorter than their
    queries, empty ones, padded batches."""
    B, H = 4, 5
    assert _two_tiles(B * H, grp * n)
    per = -(-top // P)
    kp, ks = _pools(B * per + 3, H, P, D, 1)
    vp, vs = _pools(B * per + 3, H, P, D, 2)
    table = _table(B, per, B * per + 3, 3)
    lens = torch.tensor([top, n, 0, n // 2 + 1], dtype=torch.int32, device=DEV)
    q = _q(B, H * grp, n, D, torch.bfloat16, n)
    _check(q, kp, vp, ks, vs, table, lens)
    ql = torch.tensor([n, n // 3, 3, n // 2 + 1], dtype=torch.int32, device=DEV)
    _check(q, kp, vp, ks, vs, table, lens, q_len=ql)
    _check(q, kp, vp, ks, vs, table, lens, causal=False, rotate_q=False, v_rotated=False)


def test_split_tokens():
    """So many sequences that half of the SMs are covered once: the tokens are split over two CTAs each."""
    B, H, grp, n, P = torch.cuda.get_device_properties(0).multi_processor_count // 4, 1, 4, 120, 64
    assert _two_tiles(B * H, grp * n)
    kp, ks = _pools(400, H, P, D, 4)
    vp, vs = _pools(400, H, P, D, 5)
    table = torch.randint(0, 400, (B, 24), dtype=torch.int32, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6))
    lens = torch.randint(0, 1537, (B,), dtype=torch.int32, device=DEV, generator=torch.Generator(device=DEV).manual_seed(7))
    lens[0], lens[1] = 1536, 1
    _check(_q(B, H * grp, n, D, torch.bfloat16, 8), kp, vp, ks, vs, table, lens)


def test_bad_page_and_garbage():
    """A page outside the pool is reported and left out; scales behind a sequence's end are not looked at."""
    B, H, grp, n, P = 16, 3, 2, 300, 16
    assert _two_tiles(B * H, grp * n)
    kp, ks = _pools(B * 8, H, P, D, 9)
    vp, vs = _pools(B * 8, H, P, D, 10)
    table = torch.arange(B * 8, dtype=torch.int32, device=DEV).view(B, 8)
    lens = torch.full((B,), 112, dtype=torch.int32, device=DEV)
    ks[table[:, 7].long()], vs[table[:, 7].long()] = float("nan"), float("inf")   # the last page holds no token
    q = _q(B, H * grp, n, D, torch.bfloat16, 11)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    run = lambda t: attention.attention_q8_paged(q, kp, vp, ks, vs, t, lens, status=status, causal=False)   # noqa: E731
    first = run(table)
    assert int(status.item()) == 0 and bool(first.isfinite().all())
    bad = table.clone()
    bad[5, 3] = B * 8
    got = run(bad)
    assert int(status.item()) == 1
    others = [b for b in range(B) if b != 5]
    assert torch.equal(got[others], first[others])
    keep = bad[5:6, [0, 1, 2, 4, 5, 6]]
    want, _, tol, _, _ = _reference(q[5:6], kp, vp, ks, vs, keep, torch.tensor([96]), None, False, True, True, D ** -0.5)
    half = torch.finfo(torch.bfloat16).eps / 2
    assert bool(((got[5:6].double() - want).abs() <= tol * (1 + half) + half * want.abs()).all())


def test_replayed_and_on_two_streams():
    B, H, grp, n, P = 4, 5, 4, 257, 64
    kp, ks = _pools(60, H, P, D, 12)
    vp, vs = _pools(60, H, P, D, 13)
    table = _table(B, 15, 60, 14)
    lens = torch.tensor([960, 333, 700, 257], dtype=torch.int32, device=DEV)
    qs = [_q(B, H * grp, n, D, torch.bfloat16, 15 + i) for i in range(2)]
    call = lambda i, **kw: attention.attention_q8_paged(qs[i], kp, vp, ks, vs, table, lens, **kw)   # noqa: E731
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(i))
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.empty_like(w) for w in want]
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            call(i, out=outs[i])
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i]) and torch.equal(outs[i], want[i])
