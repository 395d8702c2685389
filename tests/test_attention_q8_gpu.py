"""Attention over 8-bit pages (tq_attention_q8_paged_cuda) against the formula in float64.

Tolerance.  With exact codes the roundings are: q' to f16 (2^-12 of the row's largest element on each element
at the worst, 2^-11 of each element's value while normal), weights to f16 (2^-11 each), and fp32 sums.  A score
is off by at most ds = sm_scale * sum_d 2^-12 * max|q'| * |k_d|, a weight by the factor e^(2 ds), so an output
element by at most (2 ds + 2^-11) * sum_j p_j |v_j| (both computed here in float64 from the test's own
inputs), with 2^-14 of sum_j p_j |v_j| for the fp32 sums of up to 2^13 terms, and half a step of the output type.
A weight below f16's normal numbers is off by half its smallest step, 2^-25, of weights held as
2^6 p_j vs_j / 2^m with 2^m at most the row's largest p_j vs_j: by 2^-31 max_j(p_j vs_j) / vs_j, which is
2^-31 max_j(p_j vs_j) sum_j |code_j| of an output element (an element whose code is 0 for the one token that a
row attends to is the sum of such weights alone).
The log-sum-exp is off by at most ds + 2^-14.

That bound is for the worst signs.  The error's size is held to three times what independent roundings give: a
rounding is evenly spread over +- half a step, at most 2^-11 of the value, so its variance is at most 2^-22 / 3 of the
value's square.  Those of q' move an output by sum_d e_d q'_d c_d with c_d = sm_scale sum_j p_j k_jd (v_j - o), those
of the weights by sum_j e_j p_j v_j; to first order the squares add up, over rows and elements (the Hadamard matrix
keeps them).
"""
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


def _pools(pages, H, P, D, seed, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    code = torch.randint(-127, 128, (pages, H, P, D), dtype=torch.int8, device=DEV, generator=g)
    scale = torch.exp(spread * torch.randn(pages, H, P // 16, device=DEV, generator=g)) / 100
    return code, scale


def _table(B, per, pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[: B * per].view(B, per).to(torch.int32).to(DEV).contiguous()


def _reference(q, kp, vp, ks, vs, table, kv_len, q_len, causal, rotate_q, v_rotated, sm_scale):
    """out, lse, and the tolerances of both (before the output's own rounding), float64, and the expected square of
    the whole error."""
    B, Hq, n, D = q.shape
    H = kp.shape[1]
    grp = Hq // H
    had = _hadamard(D)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    lse = torch.full((B, Hq, n), -math.inf, dtype=torch.float64, device=DEV)
    ltol = torch.zeros_like(lse)
    square = 0.0
    for b in range(B):
        L = int(kv_len[b])
        ql = n if q_len is None else int(q_len[b])
        if L == 0 or ql == 0:
            continue
        pg = table[b].long()
        k, v = ((c[pg].double() * s[pg].double().repeat_interleave(16, -1)[..., None]).transpose(0, 1).flatten(1, 2)[:, :L]
                for c, s in ((kp, ks), (vp, vs)))
        x = q[b, :, :ql].double()
        if rotate_q:
            x = x @ had
        x = x.unflatten(0, (H, grp))
        s = sm_scale * (x @ k[:, None].transpose(-1, -2))
        ds = sm_scale * 2.0 ** -12 * x.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None, None]
        if causal:
            hide = torch.arange(L, device=DEV) > (L - ql + torch.arange(ql, device=DEV))[:, None]
            s = s.masked_fill(hide, -math.inf)
            ds = ds.masked_fill(hide, 0.0)
        e = ds.amax(-1, keepdim=True)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        o, size = p @ v[:, None], p @ v.abs()[:, None]
        square_at = 0
        t = (torch.expm1(2 * e) + 2.0 ** -11 + 2.0 ** -14) * size
        step = vs[pg].double().repeat_interleave(16, -1).transpose(0, 1).flatten(1, 2)[:, :L]
        codes = vp[pg].double().transpose(0, 1).flatten(1, 2)[:, :L].abs().sum(1)
        t = t + 2.0 ** -31 * (p * step[:, None, None]).amax(-1, keepdim=True) * codes[:, None, None]
        for h in range(H):
            for some in p[h].flatten(0, 1).split(64):
                c = sm_scale * (torch.einsum("rt,td,te->rde", some, k[h], v[h]) - (some @ k[h])[..., None] * (some @ v[h])[:, None])
                rows = slice(square_at, square_at + len(some))
                square += float((x[h].flatten(0, 1)[rows].square()[..., None] * c.square()).sum()) * 2.0 ** -22 / 3
                square += float((some.square() @ v[h].square()).sum()) * 2.0 ** -22 / 3
                square_at += len(some)
            square_at = 0
        if v_rotated:
            o, t = o @ had, t @ had.abs()   # each element of the sum may be off by its own tolerance
        out[b, :, :ql], tol[b, :, :ql] = o.flatten(0, 1), t.flatten(0, 1)
        lse[b, :, :ql] = torch.logsumexp(s, -1).flatten(0, 1)
        ltol[b, :, :ql] = (e.squeeze(-1) + 2.0 ** -14).flatten(0, 1)
    return out, lse, tol, ltol, square


def _check(q, kp, vp, ks, vs, table, kv_len, q_len=None, causal=True, rotate_q=True, v_rotated=True, sm_scale=None,
           out_dtype=None, max_kv_len=None):
    D = q.shape[-1]
    got, lse = attention.attention_q8_paged(q, kp, vp, ks, vs, table, kv_len, q_len=q_len, causal=causal, rotate_q=rotate_q,
                                            v_rotated=v_rotated, sm_scale=sm_scale, out_dtype=out_dtype, return_lse=True,
                                            max_kv_len=max_kv_len)
    want, wlse, tol, ltol, square = _reference(q, kp, vp, ks, vs, table, kv_len, q_len, causal, rotate_q, v_rotated, sm_scale or D ** -0.5)
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    assert bool((err <= tol * (1 + half) + half * want.abs() + 1e-30).all()), (err - tol).max()
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool((got[empty] == 0).all())
    assert bool(((lse.double() - wlse).abs()[~empty] <= ltol[~empty]).all())
    # 2^-14 of the output for the fp32 sums, as above
    assert float((got.double() - want).norm()) <= 3 * square ** 0.5 + (half + 2.0 ** -14) * float(want.norm()) + 1e-30
    return got, lse


def _q(B, Hq, n, D, dtype, seed, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(B, n, Hq, D, device=DEV, generator=g) * size).to(dtype).transpose(1, 2)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("grp,n", [(1, 1), (4, 1), (8, 1), (3, 1), (4, 4), (8, 5), (1, 17), (2, 40), (5, 13)])
@pytest.mark.parametrize("P,dtype", [(16, torch.bfloat16), (128, torch.float16)])
def test_matches_formula(D, grp, n, P, dtype):
    B, H = 5, 2
    top = 700
    per = -(-top // P)
    kp, ks = _pools(B * per + 3, H, P, D, 1)
    vp, vs = _pools(B * per + 3, H, P, D, 2)
    table = _table(B, per, B * per + 3, 3)
    # one token, lengths around the blocks and the warps' first turns, empty, shorter than the queries
    lens = torch.tensor([top, 1, 0, 129, 16], dtype=torch.int32, device=DEV)
    _check(_q(B, H * grp, n, D, dtype, n), kp, vp, ks, vs, table, lens)
    if n > 1:
        ql = torch.tensor([n, 1, 3, 0, n - 1], dtype=torch.int32, device=DEV)
        _check(_q(B, H * grp, n, D, dtype, n), kp, vp, ks, vs, table, lens, q_len=ql)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("grp,n,top", [(4, 32, 300), (1, 128, 128), (8, 70, 1000), (3, 111, 140), (1, 300, 700), (2, 257, 257), (16, 40, 513)])
@pytest.mark.parametrize("P,dtype", [(16, torch.bfloat16), (64, torch.float16)])
def test_prompts_match_formula(D, grp, n, top, P, dtype):
    """Prompts: row tiles with ragged ends, lengths that end inside tiles, prefixes, sequences shorter than
    their queries, empty ones, padded batches."""
    B, H = 4, 2
    per = -(-top // P)
    kp, ks = _pools(B * per + 3, H, P, D, 1)
    vp, vs = _pools(B * per + 3, H, P, D, 2)
    table = _table(B, per, B * per + 3, 3)
    lens = torch.tensor([top, n, 0, n // 2 + 1], dtype=torch.int32, device=DEV)
    q = _q(B, H * grp, n, D, dtype, n)
    _check(q, kp, vp, ks, vs, table, lens)
    ql = torch.tensor([n, n // 3, 3, n // 2 + 1], dtype=torch.int32, device=DEV)
    _check(q, kp, vp, ks, vs, table, lens, q_len=ql)
    _check(q, kp, vp, ks, vs, table, lens, causal=False, rotate_q=False, v_rotated=False)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("causal,rotate_q,v_rotated", [(False, True, True), (True, False, True), (True, True, False), (False, False, False)])
def test_options(D, causal, rotate_q, v_rotated):
    B, H, grp, n, P = 3, 2, 4, 3, 32
    kp, ks = _pools(30, H, P, D, 4)
    vp, vs = _pools(30, H, P, D, 5)
    table = _table(B, 9, 30, 6)
    lens = torch.tensor([280, 2, 33], dtype=torch.int32, device=DEV)
    _check(_q(B, H * grp, n, D, torch.float32, 7), kp, vp, ks, vs, table, lens, causal=causal, rotate_q=rotate_q,
           v_rotated=v_rotated, sm_scale=0.05, out_dtype=torch.float32)


@pytest.mark.parametrize("n", [1, 6])
def test_long_context_and_splits(n):
    B, H, grp, D, P = 2, 1, 8, 128, 256
    kp, ks = _pools(64, H, P, D, 8)
    vp, vs = _pools(64, H, P, D, 9)
    table = _table(B, 32, 64, 10)
    lens = torch.tensor([8192, 4999], dtype=torch.int32, device=DEV)
    q = _q(B, H * grp, n, D, torch.bfloat16, 11)
    a = _check(q, kp, vp, ks, vs, table, lens)
    # the planned length changes the split, not what is attended
    for most in (1, 100, 3000):
        b = _check(q, kp, vp, ks, vs, table, lens, max_kv_len=most)
        assert float((a[0].float() - b[0].float()).abs().max()) <= 2.0 ** -7 * float(a[0].float().abs().max())


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [2, 20, 130])   # rows for each of the three kernels
def test_scales_of_all_sizes(n, D):
    """Blocks whose scales differ by many orders, zero blocks (scale 0) and very large scores."""
    B, H, grp, P = 2, 2, 4, 16
    kp, ks = _pools(40, H, P, D, 12)
    vp, vs = _pools(40, H, P, D, 13, spread=6.0)
    vp[::5] = 0
    vs[::5] = 0
    kp[3::7] = 0
    ks[3::7] = 0
    table = _table(B, 20, 40, 14)
    lens = torch.tensor([320, 201], dtype=torch.int32, device=DEV)
    for size in (0.0, 1e-3, 1.0, 30.0):
        _check(_q(B, H * grp, n, D, torch.float32, 15, size), kp, vp, ks, vs, table, lens, out_dtype=torch.float32)
    # only zero values
    got = attention.attention_q8_paged(_q(B, H * grp, n, D, torch.float32, 1), kp, vp * 0, ks, vs * 0, table, lens)
    assert bool((got == 0).all())


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [3, 25, 130])
def test_garbage_behind_the_sequence_is_not_seen(n, D):
    B, H, grp, P = 2, 2, 4, 32
    kp, ks = _pools(20, H, P, D, 16)
    vp, vs = _pools(20, H, P, D, 17)
    table = _table(B, 10, 20, 18)
    lens = torch.tensor([50, 161], dtype=torch.int32, device=DEV)
    q = _q(B, H * grp, n, D, torch.bfloat16, 19)
    a = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens)
    for b in range(B):
        L = int(lens[b])
        for p in range(10):
            pg, lo = int(table[b, p]), max(0, L - p * P)
            kp[pg, :, min(lo, P):] = -128
            vp[pg, :, min(lo, P):] = 127
            first = min(-(-lo // 16), P // 16)   # scale blocks wholly behind the last token
            ks[pg, :, first:] = float("nan")
            vs[pg, :, first:] = float("inf")
        table[b, -(-L // P):] = -1
    assert torch.equal(a, attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_bad_page_is_reported_and_left_out(n, D):
    B, H, P = 1, 1, 16
    kp, ks = _pools(8, H, P, D, 20)
    vp, vs = _pools(8, H, P, D, 21)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    lens = torch.tensor([128], dtype=torch.int32, device=DEV)
    q = _q(B, 2, n, D, torch.float32, 22)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    run = lambda t: attention.attention_q8_paged(q, kp, vp, ks, vs, t, lens, status=status, causal=False)   # noqa: E731
    run(table)
    assert int(status.item()) == 0
    bad = table.clone()
    bad[0, 3] = 8
    bad[0, 7] = -1
    got = run(bad)
    assert int(status.item()) == 1
    keep = torch.tensor([[0, 1, 2, 4, 5, 6]], dtype=torch.int32, device=DEV)
    want, _, tol, _, _ = _reference(q, kp, vp, ks, vs, keep, torch.tensor([96]), None, False, True, True, D ** -0.5)
    assert bool(((got.double() - want).abs() <= tol + 1e-6).all())


def test_strides_single_token_form_and_outputs():
    B, Hq, H, n, D, P = 2, 6, 2, 4, 128, 16
    kp, ks = _pools(20, H, P, D, 23)
    vp, vs = _pools(20, H, P, D, 24)
    table = _table(B, 10, 20, 25)
    lens = torch.tensor([150, 77], dtype=torch.int32, device=DEV)
    qkv = torch.randn(B, n, Hq + 2 * H, D, device=DEV).half()
    q = qkv[:, :, :Hq].transpose(1, 2)
    want = attention.attention_q8_paged(q.contiguous(), kp, vp, ks, vs, table, lens)
    assert torch.equal(attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens), want)
    out = torch.full((B, Hq, n, D), 5.0, device=DEV).half()
    lse = torch.empty(B, Hq, n, device=DEV)
    assert attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, out=out, lse_out=lse).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    one, l1 = attention.attention_q8_paged(q[:, :, 0], kp, vp, ks, vs, table, lens, return_lse=True)
    four, l4 = attention.attention_q8_paged(q[:, :, :1], kp, vp, ks, vs, table, lens, return_lse=True)
    assert one.shape == (B, Hq, D) and l1.shape == (B, Hq) and torch.equal(one, four.squeeze(2)) and torch.equal(l1, l4.squeeze(2))
    assert attention.attention_q8_paged(q[:, :, :0], kp, vp, ks, vs, table, lens).shape == (B, Hq, 0, D)
    assert attention.attention_q8_paged(q[:0], kp, vp, ks, vs, table[:0], lens[:0]).shape == (0, Hq, n, D)


def test_two_streams_and_graph_replay():
    B, H, grp, D, P = 2, 2, 8, 128, 64
    kp, ks = _pools(80, H, P, D, 26)
    vp, vs = _pools(80, H, P, D, 27)
    table = _table(B, 40, 80, 28)
    lens = torch.tensor([2500, 1333], dtype=torch.int32, device=DEV)
    qs = [_q(B, H * grp, 1, D, torch.bfloat16, 30 + i) for i in range(2)]
    want = [attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(attention.attention_q8_paged(qs[i], kp, vp, ks, vs, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want[0])
    with torch.cuda.graph(graph):
        attention.attention_q8_paged(qs[0], kp, vp, ks, vs, table, lens, out=out, max_kv_len=2560)
    for L in (2500, 17, 0, 2560):
        lens.fill_(L)
        graph.replay()
        assert torch.equal(out, attention.attention_q8_paged(qs[0], kp, vp, ks, vs, table, lens, max_kv_len=2560))


def test_append_then_attend_with_rotary():
    """The three operators as a serving step runs them, against attention on the unquantized rows: prompt pieces
    and single tokens of a padded batch."""
    B, Hq, H, D, P = 3, 8, 2, 128, 16
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    table = _table(B, 12, 40, 31)
    kp, vp = (torch.zeros(40, H, P, D, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(40, H, 1, device=DEV) for _ in range(2))
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    held = [[] for _ in range(B)]
    for step, (n, new) in enumerate([(60, [60, 9, 31]), (1, [1, 1, 1]), (1, [1, 0, 1]), (5, [5, 5, 2]), (50, [3, 50, 0]), (1, [1, 1, 1])]):
        g = torch.Generator(device=DEV).manual_seed(step)
        x = torch.randn(B, n, Hq + 2 * H, D, device=DEV, generator=g).bfloat16()
        q, k, v = (t.transpose(1, 2) for t in x.split([Hq, H, H], dim=2))
        new_t = torch.tensor(new, dtype=torch.int32, device=DEV)
        slots = (pos[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)).contiguous()
        kr = ops.rotary(k.float().contiguous(), slots, rope)
        qr = ops.kv_append_rotary_paged(k, v, kp, vp, table, pos, rope=rope, q=q, new_len=new_t, k_scale=ks, v_scale=vs)
        pos += new_t
        out = attention.attention_q8_paged(qr, kp, vp, ks, vs, table, pos, q_len=new_t)
        for b in range(B):
            held[b].append((kr[b, :, :new[b]], v[b, :, :new[b]].float()))
            K, V = (torch.cat(t, 1).double().repeat_interleave(Hq // H, 0) for t in zip(*held[b]))
            L = K.shape[1]
            s = qr[b, :, :new[b]].double() @ K.transpose(1, 2) / math.sqrt(D)
            hide = torch.arange(L, device=DEV) > (L - new[b] + torch.arange(new[b], device=DEV))[:, None]
            want = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ V
            if new[b]:
                # 8-bit codes of rotated rows: a step is the block's maximum / 127, about 4.5 / 127 deviations, its
                # error 0.29 steps (0.01 deviations) on values and, over sqrt(D) scaled sums, on scores
                rel = float((out[b, :, :new[b]].double() - want).norm() / want.norm())
                assert rel < 0.03, rel
            assert bool((out[b, :, new[b]:] == 0).all())


def test_bound_of_the_lengths():
    """A sequence longer than max_kv_len: reported where the work memory is sized by it (many rows)."""
    B, H, grp, D, P, n = 2, 1, 8, 128, 64, 64
    kp, ks = _pools(32, H, P, D, 1)
    vp, vs = _pools(32, H, P, D, 2)
    table = _table(B, 16, 32, 3)
    lens = torch.tensor([700, 900], dtype=torch.int32, device=DEV)
    q = _q(B, H * grp, n, D, torch.bfloat16, 4)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, status=status)
    got = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, max_kv_len=900, status=status)
    assert int(status.item()) == 0 and torch.equal(got, want)
    got = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, max_kv_len=800, status=status)
    assert int(status.item()) == 1 and torch.equal(got[0], want[0])


@pytest.mark.parametrize("n", [1, 8, 64])
def test_prompts_on_two_streams_and_replayed(n):
    """Each call has work memory of its own: overlapping calls and two graphs replayed in turn keep their results."""
    B, H, grp, D, P = 3, 2, 8, 128, 64
    kp, ks = _pools(60, H, P, D, 36)
    vp, vs = _pools(60, H, P, D, 37)
    table = _table(B, 20, 60, 38)
    lens = torch.tensor([1280, 333, 700], dtype=torch.int32, device=DEV)
    qs = [_q(B, H * grp, n, D, torch.bfloat16, 40 + i) for i in range(2)]
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


def test_refusals():
    B, H, D, P = 2, 2, 128, 16
    kp, ks = _pools(8, H, P, D, 1)
    vp, vs = _pools(8, H, P, D, 2)
    table = _table(B, 4, 8, 1)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    q = _q(B, 4, 2, D, torch.float16, 1)
    good = dict(q=q, k_pool=kp, v_pool=vp, k_scale=ks, v_scale=vs, page_table=table, kv_len=lens)
    attention.attention_q8_paged(**good)
    for change in (dict(q=q.double()), dict(q=q[:, :3]), dict(q=q[..., :64]), dict(k_pool=kp.float()), dict(v_pool=vp[:4]),
                   dict(k_scale=ks.half()), dict(v_scale=vs[:, :1]), dict(page_table=table.long()), dict(kv_len=lens.long()),
                   dict(kv_len=lens[:1]), dict(q_len=lens[:1]), dict(out=torch.zeros(B, 4, 2, 64, device=DEV)),
                   dict(lse_out=lens), dict(status=lens.float()), dict(q=q.cpu()), dict(k_pool=kp.cpu()), dict(kv_len=lens.cpu())):
        with pytest.raises(ValueError):
            attention.attention_q8_paged(**{**good, **change})
    wide = torch.zeros(B, 4, 2, D + 4, dtype=torch.float16, device=DEV)
    for change in (dict(q=wide[..., :D]), dict(max_kv_len=65), dict(max_kv_len=-1), dict(sm_scale=float("nan"))):
        with pytest.raises(ops.L.TQError):
            attention.attention_q8_paged(**{**good, **change})
