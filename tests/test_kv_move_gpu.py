"""Moving rows of paged caches (tq_kv_move_paged_cuda): TurboQuant rows as bytes, 8-bit rows against the rule in float32, whose
operations (a product, a quotient, rounding to the nearest whole number) are the same on both sides, so that codes and scales are equal."""
import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BYTES = {2: 10, 3: 14, 4: 18}


def _pools(bits, pages, H, P, D, seed, alike=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if bits == 8:
        out = []
        for _ in range(2):
            code = torch.randint(-127, 128, (pages, H, P, D), dtype=torch.int8, device=DEV, generator=g)
            quiet = torch.rand(pages, H, P, 1, device=DEV, generator=g) < 0.3      # rows well below their block's largest
            code = torch.where(quiet, code // 9, code)
            scale = torch.exp(torch.randn(pages, H, P // 16, device=DEV, generator=g)) / 100
            if alike:
                scale = torch.where(torch.rand(scale.shape, device=DEV, generator=g) < 0.8, 0.125, scale)
            out += [code, scale]
        return out
    rand = lambda b: torch.randint(0, 256, (pages, H, P, D // 32, b), dtype=torch.uint8, device=DEV, generator=g)   # noqa: E731
    return [rand(BYTES[bits]), None, rand(18), None]


def _expected(pool, scale, w, table, to_table, src, first, count, in_place):
    """Pool, scale and weights after the move, and the number of rows left."""
    old, new = pool, pool.clone()
    s_new, w_new = (None if t is None else t.clone() for t in (scale, w))
    N, H, P = pool.shape[:3]
    B, m = src.shape[0], src.shape[-1]
    src3 = src if src.dim() == 3 else src[:, None].expand(B, H, m)
    src3, tab, to_tab = src3.cpu().tolist(), table.cpu().tolist(), to_table.cpu().tolist()
    left = 0
    at = lambda rows, s: (rows[s // P], s % P) if 0 <= s < len(rows) * P and 0 <= rows[s // P] < N else None   # noqa: E731
    for b in range(B):
        f = min(max(first[b], 0), len(to_tab[b]) * P)
        c = min(max(count[b], 0), m)
        for h in range(H):
            blocks = {}
            for j in range(c):
                s = src3[b][h][j]
                if s < 0:
                    continue
                a, d = at(tab[b], s), at(to_tab[b], f + j)
                if a is None or d is None or (in_place and s < f + j):
                    left += 1
                    continue
                blocks.setdefault((f + j) // 16, []).append((a, d))
                if w is not None:
                    w_new[d[0], h, d[1]] = w[a[0], h, a[1]]
                if scale is None:
                    new[d[0], h, d[1]] = old[a[0], h, a[1]]
            if scale is None:
                continue
            for block, rows in blocks.items():
                older = [(at(to_tab[b], s),) * 2 for s in range(block * 16, (block + 1) * 16) if s < f]
                if all(a == d for a, d in rows):
                    continue
                both = older + rows
                pa, sa = (torch.tensor([a[i] for a, _ in both], device=DEV) for i in (0, 1))
                pd, sd = (torch.tensor([d[i] for _, d in both], device=DEV) for i in (0, 1))
                code, size = old[pa, h, sa].float(), scale[pa, h, sa // 16]
                if bool((size == size[0]).all()):
                    now, fresh = size[0], code
                else:
                    now = (code.abs().amax(-1) * size * (torch.ones((), device=DEV) / 127)).amax()
                    fresh = torch.round(code * (size / now)[:, None]).clamp(-127, 127)
                new[pd, h, sd] = fresh.to(torch.int8)
                s_new[pd[0], h, sd[0] // 16] = now
    return new, s_new, w_new, left


def _check(bits, B, H, D, P, src, pages, first=None, count=None, weights=False, to=None, seed=0, alike=False, table=None):
    per = pages
    kp, ks, vp, vs = _pools(bits, B * per * 2 + 1, H, P, D, seed, alike)
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(B * per * 2 + 1, generator=g).to(torch.int32).to(DEV)
    if table is None:
        table = order[: B * per].view(B, per).contiguous()
    to_table = order[B * per: 2 * B * per].view(B, per).contiguous() if to else table
    w = torch.rand(kp.shape[:3], device=DEV) if weights else None
    src = src.to(torch.int32).to(DEV).contiguous()
    f = [0] * B if first is None else first
    c = [src.shape[-1]] * B if count is None else count
    want = [_expected(p, s, w if i == 0 else None, table, to_table, src, f, c, not to) for i, (p, s) in enumerate(((kp, ks), (vp, vs)))]
    over, status = (torch.zeros(1, dtype=torch.int32, device=DEV) for _ in range(2))
    ops.kv_move_paged(kp, vp, table, src, first=None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV),
                      count=None if count is None else torch.tensor(count, dtype=torch.int32, device=DEV), k_scale=ks, v_scale=vs,
                      weights=w, to_table=to_table if to else None, overflow=over, status=status)
    for (p, s), (wp, ws, ww, _) in zip(((kp, ks), (vp, vs)), want):
        assert torch.equal(p, wp)
        assert s is None or torch.equal(s, ws)
        assert ww is None or torch.equal(w, ww)
    assert int(over) == want[0][3] and int(status) == 0


def _kept(B, H, top, m, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.stack([torch.stack([torch.randperm(top, generator=g)[:m].sort().values for _ in range(H)]) for _ in range(B)])


@pytest.mark.parametrize("bits", [8, 2, 3, 4])
@pytest.mark.parametrize("D,P,top,m", [(128, 16, 40, 9), (128, 32, 300, 150), (256, 16, 300, 64), (256, 64, 500, 333), (128, 16, 65, 65)])
def test_kept_tokens_move_to_the_front(bits, D, P, top, m):
    _check(bits, 2, 2, D, P, _kept(2, 2, top, m, m), -(-top // P), weights=True, seed=m)


@pytest.mark.parametrize("bits", [8, 3])
@pytest.mark.parametrize("D", [128, 256])
def test_accepted_paths(bits, D):
    # behind caches that end at all places of a block; paths from no node to all of them
    first = [0, 5, 15, 16, 31, 40]
    count = [4, 0, 7, 1, 6, 3]
    src = torch.tensor([[0, 2, 5, 6, -1, -1, -1], [0, 0, 0, 0, 0, 0, 0], [0, 1, 2, 3, 4, 5, 6], [3, -1, -1, -1, -1, -1, -1],
                        [1, 4, 9, 15, 20, 24, 25], [2, 3, 8, -1, -1, -1, -1]])
    src = torch.where(src >= 0, src + torch.tensor(first)[:, None], -1)
    _check(bits, 6, 2, D, 16, src, 5, first=first, count=count, seed=D)
    _check(bits, 6, 2, D, 16, src, 5, first=first, count=count, seed=D, to=True)


@pytest.mark.parametrize("bits", [8, 4])
def test_many_chunks_in_place(bits):
    """Chunks that read what other chunks write: everything moves down by a few slots, or by many."""
    for shift in (1, 17, 64, 100):
        m = 1500
        src = (torch.arange(m) + shift).expand(2, 2, m)
        _check(bits, 2, 2, 128, 64, src, -(-(m + shift) // 64), weights=True, seed=shift)
    _check(bits, 1, 1, 128, 16, _kept(1, 1, 6000, 3100, 1), 375, seed=9)


@pytest.mark.parametrize("bits", [8, 2])
def test_other_pages(bits):
    _check(bits, 2, 2, 128, 32, _kept(2, 2, 300, 130, 1), 10, weights=True, to=True, seed=1)
    # any order, up and down, the same row twice
    g = torch.Generator().manual_seed(2)
    _check(bits, 2, 2, 128, 32, torch.randint(0, 300, (2, 2, 130), generator=g), 10, first=[3, 64], weights=True, to=True, seed=2)


def test_rows_of_one_scale_keep_codes_and_scale():
    _check(8, 2, 2, 128, 32, _kept(2, 2, 300, 130, 1), 10, seed=1, alike=True)


def test_any_order_in_place():
    """Rows that move down in any order, and the same row to several places."""
    g = torch.Generator().manual_seed(5)
    src = torch.arange(200) + torch.randint(0, 90, (2, 2, 200), generator=g)
    _check(8, 2, 2, 128, 16, src, 19, seed=4)
    _check(3, 2, 2, 128, 16, src, 19, seed=4)


@pytest.mark.parametrize("bits", [8, 3])
def test_rows_without_a_place_are_left_and_counted(bits):
    H = 2
    src = torch.tensor([[[4, 3, 1, 90, 79, 1 << 30, -7, 20], [5, 6, 7, 8, 9, 10, 11, 12]]])   # capacity 80; 3 -> 1 is down, 1 -> 2 up
    _check(bits, 1, H, 128, 16, src, 5, first=[0], seed=1)
    _check(bits, 1, H, 128, 16, src, 5, first=[77], seed=1)            # destinations behind the capacity
    _check(bits, 1, H, 128, 16, src, 5, first=[1 << 30], seed=1)
    _check(bits, 1, H, 128, 16, src, 5, first=[-4], count=[1000], seed=1)
    _check(bits, 1, H, 128, 16, src, 5, count=[-1], seed=1)
    table = torch.tensor([[0, -1, 11, 3, 4]], dtype=torch.int32, device=DEV)    # 11 pages: 11 is outside
    wide = torch.arange(64).expand(1, H, 64) + 14
    _check(bits, 1, H, 128, 16, wide, 5, seed=2, table=table)
    _check(bits, 1, H, 128, 16, wide, 5, seed=2, table=table, to=True)


def test_eviction_keeps_what_the_kept_tokens_hold():
    """8-bit values after a move are within half a step of the block's new scale of those before."""
    B, H, D, P, top, m = 2, 4, 128, 32, 500, 200
    kp, ks, vp, vs = _pools(8, 40, H, P, D, 3)
    table = torch.arange(32, dtype=torch.int32, device=DEV).view(2, 16)
    src = _kept(B, H, top, m, 4).to(torch.int32).to(DEV)
    before = ops.dequantize_q8(kp, ks).double()[table.long()].transpose(1, 2).flatten(2, 3)
    want = before.gather(2, src.long()[..., None].expand(-1, -1, -1, D))
    ops.kv_move_paged(kp, vp, table, src, k_scale=ks, v_scale=vs)
    after = ops.dequantize_q8(kp, ks).double()[table.long()].transpose(1, 2).flatten(2, 3)[:, :, :m]
    step = ks.double()[table.long()].transpose(1, 2).flatten(2, 3).repeat_interleave(16, -1)[:, :, :m, None]
    # half a step, codes of the largest row rounded from 127 +- 2^-22, products in float32 and the value's own rounding
    assert bool(((after - want).abs() <= step * (0.5 + 2.0 ** -14)).all())


def test_refusals():
    kp, ks, vp, vs = _pools(8, 8, 2, 16, 128, 1)
    t3, _, t4, _ = _pools(3, 8, 2, 16, 128, 1)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    src = torch.zeros(1, 2, 3, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    good = dict(k_pool=kp, v_pool=vp, page_table=table, src=src, k_scale=ks, v_scale=vs)
    ops.kv_move_paged(**good)
    ops.kv_move_paged(t3, t4, table, src)
    for change in (dict(src=src.long()), dict(src=src[:, :1].expand(1, 3, 3).contiguous()), dict(src=src[0]), dict(src=src.expand(2, 2, 3)),
                   dict(first=one.long()), dict(first=one.expand(2)), dict(count=one.float()), dict(k_scale=None), dict(v_scale=vs[:4]),
                   dict(v_pool=vp[:4]), dict(weights=torch.zeros(8, 2, 8, device=DEV)), dict(weights=torch.zeros(8, 2, 16)),
                   dict(to_table=table.long()), dict(to_table=table.expand(2, 8)), dict(overflow=one.float()), dict(k_pool=t3), dict(k_pool=kp.cpu()),
                   dict(k_pool=t3, v_pool=t3, k_scale=None, v_scale=None), dict(k_pool=t3, v_pool=t4)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.kv_move_paged(**{**good, **change})
    assert attention.last_status() == 0
