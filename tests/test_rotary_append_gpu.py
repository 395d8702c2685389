"""The paged append with the rotation on the way (tq_kv_append_rotary_paged_cuda).

TQ pages must hold, byte for byte, what rotation in float32 followed by the paged append writes.  8-bit pages
are compared with a plain restatement on the same float32 rows (equal codes and scales), and their values
with the rows: a code is off by at most half a step when written, and by at most half a step more each time
the block's scale grew.
"""
import pytest
import torch

from leankv_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _step(B, n, hq, hk, D, dtype, seed):
    """q, k, v views of one projection's output."""
    x = torch.randn(B, n, hq + 2 * hk, D, device=DEV, generator=_gen(seed)).to(dtype)
    x[..., 5] *= 12
    return tuple(t.transpose(1, 2) for t in x.split([hq, hk, hk], dim=2))


def _table(B, per, spare, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(B * per + spare, generator=g)[: B * per].view(B, per).to(torch.int32).to(DEV).contiguous()


def _turned(k, rope, positions):
    return ops.rotary(k.float().contiguous(), positions, rope)


@pytest.mark.parametrize("D,kt,P,dtype,axes,interleaved,R", [
    (128, 3, 16, torch.bfloat16, 1, False, 128), (128, 4, 64, torch.float16, 3, False, 128),
    (128, 2, 32, torch.float32, 1, True, 64), (256, 4, 32, torch.bfloat16, 1, False, 256),
    (256, 3, 16, torch.float32, 3, True, 128), (256, 2, 128, torch.float16, 1, False, 48)])
def test_tq_pages_equal_rotation_then_append(D, kt, P, dtype, axes, interleaved, R):
    B, hq, hk, per = 4, 6, 2, 5
    rope = ops.Rotary(ops.rotary_frequencies(R, device=DEV),
                      ops.rotary_axes((R // 8, R // 8, R // 4), DEV) if axes == 3 else None, interleaved)
    table = _table(B, per, 3, P)
    pages = B * per + 3
    kb = ops.BLOCK_BYTES[kt]
    kp = torch.randint(0, 255, (pages, hk, P, D // 32, kb), dtype=torch.uint8, device=DEV, generator=_gen(1))
    vp = torch.randint(0, 255, (pages, hk, P, D // 32, 18), dtype=torch.uint8, device=DEV, generator=_gen(2))
    kw, vw = kp.clone(), vp.clone()
    for seed, (n, pos, new) in enumerate([(1, [0, 15, 16, 40], None), (1, [7, 0, 33, 17], [1, 0, 1, 1]),
                                          (37, [0, 5, 16, 30], [37, 20, 1, 0]), (2, [15, 14, 31, 3], None),
                                          (16, [0, 1, 16, 8], [16, 16, 15, 3])]):
        q, k, v = _step(B, n, hq, hk, D, dtype, seed)
        pos_t = torch.tensor(pos, dtype=torch.int32, device=DEV)
        new_t = None if new is None else torch.tensor(new, dtype=torch.int32, device=DEV)
        slots = (pos_t[:, None] + torch.arange(n, device=DEV, dtype=torch.int32)).contiguous()
        positions = None
        if axes == 3:
            positions = torch.randint(0, 100000, (3, B, n), dtype=torch.int32, device=DEV, generator=_gen(seed))
        got = ops.kv_append_rotary_paged(k, v, kp, vp, table, pos_t, rope=rope, positions=positions, q=q, new_len=new_t)
        where = slots if positions is None else positions
        assert torch.equal(got, ops.rotary(q, where, rope))
        kt32 = _turned(k, rope, where)
        for b in range(B):
            m = n if new is None else new[b]
            if not m:
                continue
            one, at = table[b:b + 1].contiguous(), pos_t[b:b + 1].contiguous()
            ops.kv_append_paged(kt32[b:b + 1, :, :m].contiguous(), kw, one, at, qtype=kt)
            ops.kv_append_paged(v[b:b + 1, :, :m].contiguous(), vw, one, at, qtype=4)
        assert torch.equal(kp, kw) and torch.equal(vp, vw), seed


def test_tq_pages_without_rotation_or_hadamard():
    B, hk, D, P = 2, 3, 128, 16
    table = _table(B, 4, 0, 1)
    _, k, v = _step(B, 20, 1, hk, D, torch.float16, 4)
    pos = torch.tensor([3, 12], dtype=torch.int32, device=DEV)
    a, b = (torch.zeros(8, hk, P, 4, n, dtype=torch.uint8, device=DEV) for n in (14, 18))
    c, d = a.clone(), b.clone()
    assert ops.kv_append_rotary_paged(k, v, a, b, table, pos, rotate=False) is None
    ops.kv_append_paged(k.contiguous(), c, table, pos, qtype=3, rotate=False)
    ops.kv_append_paged(v.contiguous(), d, table, pos, qtype=4, rotate=False)
    assert torch.equal(a, c) and torch.equal(b, d)


def _append8_plain(code, scale, rows, table, pos, new, P):
    """The 8-bit append restated on float32 rows [B, H, n, D] (already rotated), in place."""
    for b in range(rows.shape[0]):
        lo, hi = int(pos[b]), int(pos[b]) + int(new[b])
        for first in range(lo // 16 * 16, hi if hi > lo else 0, 16):
            if first // P >= table.shape[1] or first < 0:
                continue
            page, off = int(table[b, first // P]), first % P
            if not 0 <= page < code.shape[0]:
                continue
            a, e = max(lo, first), min(hi, first + 16)
            x = rows[b, :, a - lo:e - lo]
            old = scale[page, :, off // 16] if a > first else torch.zeros(rows.shape[1], device=DEV)
            s = torch.maximum(old, x.abs().amax((-1, -2)) * (1.0 / 127.0))
            s = torch.where(s >= 2.0 ** -100, s, torch.zeros_like(s))
            inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))[:, None, None]
            if a > first:
                c = code[page, :, off:off + a - first]
                c.copy_(torch.where((old < s)[:, None, None], torch.round(c.float() * (old[:, None, None] * inv)), c.float()).to(torch.int8))
            code[page, :, off + a - first:off + e - first] = torch.round(x * inv).clamp(-127, 127).to(torch.int8)
            scale[page, :, off // 16] = s


@pytest.mark.parametrize("D,P,dtype", [(128, 16, torch.bfloat16), (256, 32, torch.float16), (128, 128, torch.float32),
                                       (256, 16, torch.float32)])
def test_q8_pages_equal_restatement(D, P, dtype):
    B, hq, hk, per = 4, 4, 2, 160 // P + 1
    pages = B * per + 2
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    table = _table(B, per, 2, P)
    kp, vp = (torch.randint(-127, 128, (pages, hk, P, D), dtype=torch.int8, device=DEV, generator=_gen(s)) for s in (1, 2))
    ks, vs = (torch.rand(pages, hk, P // 16, device=DEV, generator=_gen(s)) for s in (3, 4))
    kw, vw, ksw, vsw = kp.clone(), vp.clone(), ks.clone(), vs.clone()
    pos = torch.tensor([0, 5, 16, 31], dtype=torch.int32, device=DEV)
    for seed, (n, new, size) in enumerate([(40, [40, 17, 1, 0], 1.0), (1, None, 1.0), (1, None, 3.0), (1, [1, 0, 1, 1], 0.1),
                                           (5, [5, 4, 0, 2], 30.0), (16, None, 0.0), (33, [3, 33, 20, 16], 100.0)]):
        q, k, v = _step(B, n, hq, hk, D, dtype, seed)
        k, v = k * size, v * size
        new_t = None if new is None else torch.tensor(new, dtype=torch.int32, device=DEV)
        slots = (pos[:, None] + torch.arange(n, device=DEV, dtype=torch.int32)).contiguous()
        got = ops.kv_append_rotary_paged(k, v, kp, vp, table, pos, rope=rope, q=q, new_len=new_t, k_scale=ks, v_scale=vs)
        assert torch.equal(got, ops.rotary(q, slots, rope))
        count = torch.full((B,), n, device=DEV) if new is None else new_t
        kr = ops.hadamard_(_turned(k, rope, slots).contiguous(), D)
        vr = ops.hadamard_(v.float().contiguous(), D)
        _append8_plain(kw, ksw, kr, table, pos, count, P)
        _append8_plain(vw, vsw, vr, table, pos, count, P)
        assert torch.equal(ks, ksw) and torch.equal(vs, vsw), seed
        assert torch.equal(kp, kw) and torch.equal(vp, vw), seed
        if new is None or min(new) > 0:
            values = ops.dequantize_q8(kp, ks)
            for b in range(B):
                s = slots[b, :int(count[b])].long()
                step = ksw[table[b].long()[s // P], :, s % P // 16].T[..., None]
                # half a step, and the roundings of 1 / s and of the two products
                err = (values[table[b].long()[s // P], :, s % P].transpose(0, 1) - kr[b, :, :len(s)]).abs()
                assert bool((err <= step * (0.5 + 130 * 3 * 2.0 ** -24)).all())
        pos += count.to(torch.int32)


def test_q8_values_within_half_a_step_of_64_bits():
    """A written row against the rotation and the Hadamard matrix in 64 bits."""
    B, hk, n, D, P = 2, 2, 48, 128, 16
    _, k, v = _step(B, n, 1, hk, D, torch.bfloat16, 9)
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    table = _table(B, 3, 0, 1)
    kp, vp = (torch.zeros(6, hk, P, D, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(6, hk, 1, device=DEV) for _ in range(2))
    ops.kv_append_rotary_paged(k, v, kp, vp, table, None, rope=rope, k_scale=ks, v_scale=vs)
    i = torch.arange(D, device=DEV)
    odd = torch.zeros(D, D, device=DEV, dtype=torch.int64)
    for bit in range(7):
        odd ^= ((i[:, None] & i) >> bit) & 1
    had = (1 - 2 * odd).double() / D ** 0.5
    angle = torch.arange(n, device=DEV).double()[:, None] * rope.inv_freq
    a, b = k.double()[..., :64], k.double()[..., 64:]
    kr = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1) @ had
    for codes, scale, rows in ((kp, ks, kr), (vp, vs, v.double() @ had)):
        values = ops.dequantize_q8(codes, scale, torch.float32)[table.long()].transpose(1, 2).flatten(2, 3).double()
        step = scale[table.long()].transpose(1, 2).flatten(2, 3).repeat_interleave(16, -1)[..., None].double()
        top = rows.abs().amax().item()
        # half a step; the float32 rows are off by at most 11 roundings (angle, 3 of the turn, 7 stages) of sums
        # whose terms are at most sqrt(D) times the largest row value; the value's product is rounded once
        tol = step * (0.5 + 127 * 4 * 2.0 ** -24) + 11 * 2.0 ** -24 * top * D ** 0.5
        assert bool(((values - rows).abs() <= tol).all())


def test_rows_without_a_place_are_counted():
    B, hk, D, P = 3, 2, 128, 16
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    table = torch.tensor([[0, 1], [-1, 2], [3, 99]], dtype=torch.int32, device=DEV)
    q, k, v = _step(B, 30, 2, hk, D, torch.float16, 3)
    pos = torch.tensor([8, 4, 2], dtype=torch.int32, device=DEV)   # 6 rows of sequence 0 lie behind its pages
    lost = (6 + 12 + 16) * hk * 2
    for kind in (3, 8):
        over = torch.zeros(1, dtype=torch.int32, device=DEV)
        if kind == 8:
            kp, vp = (torch.full((4, hk, P, D), 7, dtype=torch.int8, device=DEV) for _ in range(2))
            ks, vs = (torch.ones(4, hk, 1, device=DEV) for _ in range(2))
            ops.kv_append_rotary_paged(k, v, kp, vp, table, pos, rope=rope, q=q, k_scale=ks, v_scale=vs, overflow=over)
            # the slots before each sequence's first row belong to earlier rows, rescaled or not; page 2 is
            # sequence 1's second page: slots 16 .. 33 of which rows 12 .. 29 fill 16
            assert not torch.equal(kp[2], torch.full_like(kp[2], 7))
        else:
            kp = torch.zeros(4, hk, P, 4, 14, dtype=torch.uint8, device=DEV)
            vp = torch.zeros(4, hk, P, 4, 18, dtype=torch.uint8, device=DEV)
            ops.kv_append_rotary_paged(k, v, kp, vp, table, pos, rope=rope, q=q, overflow=over)
            assert bool((kp[0, :, :8] == 0).all())
        # sequence 1: 12 rows on the page that is not there and 2 behind its two pages
        assert int(over.item()) == lost + 2 * hk * 2


def test_append_graph_replay():
    B, hq, hk, D, P = 2, 4, 2, 128, 16
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    table = _table(B, 4, 0, 5)
    q, k, v = _step(B, 1, hq, hk, D, torch.bfloat16, 3)
    pools = [torch.zeros(8, hk, P, D, dtype=torch.int8, device=DEV) for _ in range(4)]
    scales = [torch.zeros(8, hk, 1, device=DEV) for _ in range(4)]
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv_append_rotary_paged(k, v, pools[0], pools[1], table, pos, rope=rope, q=q, q_out=out, k_scale=scales[0], v_scale=scales[1])
    for t in range(40):
        k.copy_(torch.randn(k.shape, device=DEV, generator=_gen(t)))
        v.copy_(torch.randn(v.shape, device=DEV, generator=_gen(100 + t)))
        pos.fill_(t)
        graph.replay()
        want = ops.kv_append_rotary_paged(k, v, pools[2], pools[3], table, pos, rope=rope, q=q, k_scale=scales[2], v_scale=scales[3])
        assert torch.equal(out, want)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    assert torch.equal(scales[0], scales[2]) and torch.equal(scales[1], scales[3])


def test_dequantize_q8_types():
    codes = torch.randint(-127, 128, (3, 2, 32, 256), dtype=torch.int8, device=DEV, generator=_gen(1))
    scale = torch.rand(3, 2, 2, device=DEV, generator=_gen(2)) + 0.01
    want = codes.float() * scale.repeat_interleave(16, -1)[..., None]
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        assert torch.equal(ops.dequantize_q8(codes, scale, dtype), want.to(dtype))
    assert ops.dequantize_q8(codes[:0], scale[:0]).shape == (0, 2, 32, 256)


def test_append_refusals():
    B, hk, D, P = 2, 2, 128, 16
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    q, k, v = _step(B, 4, 4, hk, D, torch.float16, 1)
    table = _table(B, 2, 0, 1)
    i8 = torch.zeros(4, hk, P, D, dtype=torch.int8, device=DEV)
    sc = torch.zeros(4, hk, 1, device=DEV)
    good = dict(k=k, v=v, k_pool=i8, v_pool=i8.clone(), page_table=table, rope=rope, k_scale=sc, v_scale=sc.clone())
    ops.kv_append_rotary_paged(**good)
    tq = torch.zeros(4, hk, P, 4, 18, dtype=torch.uint8, device=DEV)
    for change in (dict(v=v[:, :1]), dict(v=v.float()), dict(k=k.double(), v=v.double()), dict(k_scale=None),
                   dict(k_scale=sc[:, :, :0]), dict(v_scale=sc.double()), dict(v_pool=tq), dict(k_pool=tq),
                   dict(k_pool=i8[:, :, ::2]), dict(page_table=table.long()), dict(page_table=table[:1]),
                   dict(pos=torch.zeros(B, device=DEV)), dict(new_len=torch.zeros(3, dtype=torch.int32, device=DEV)),
                   dict(q=q, rope=None), dict(q=q[:, :, :2]), dict(q_out=q), dict(rope=None, positions=table[:, :2]),
                   dict(positions=torch.zeros(B, 5, dtype=torch.int32, device=DEV)), dict(k=k.cpu()),
                   dict(k_pool=tq, v_pool=tq)):
        with pytest.raises(ValueError):
            ops.kv_append_rotary_paged(**{**good, **change})
    odd = torch.zeros(4, hk, 24, D, dtype=torch.int8, device=DEV)
    os = torch.zeros(4, hk, 1, device=DEV)
    for change in (dict(k_pool=odd, v_pool=odd.clone(), k_scale=os, v_scale=os.clone()),       # page size 24
                   dict(rope=ops.Rotary(ops.rotary_frequencies(256, device=DEV)))):            # wider than the head
        with pytest.raises(ops.L.TQError):
            ops.kv_append_rotary_paged(**{**good, **change})
    small = torch.zeros(4, hk, P, 64, dtype=torch.int8, device=DEV)
    with pytest.raises(ops.L.TQError):   # head_dim 64
        ops.kv_append_rotary_paged(k[..., :64], v[..., :64], small, small.clone(), table, k_scale=sc, v_scale=sc.clone())
