"""PagedKVCache with trees of drafted tokens and eviction, the operators as a serving loop runs them one after another:
append with rotation, attention, accepted paths, observed weights, eviction, steps after it.

Where outputs are compared with float64, keys and values are the ones that the pages hold (dequantized), so the tolerance is the
attention kernels' own: 2e-3 of the norm covers bfloat16's 2^-9 relative rounding error (evenly spread: 2^-9 / sqrt(3) of the norm) and the
products' f16 roundings, which the operators' own tests derive (2.8e-4 of the norm)."""
import math

import pytest
import torch

from leankv_b200 import attention, ops
from leankv_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
D, H, GRP = 128, 2, 4


def _hadamard():
    i = torch.arange(D, device=DEV)
    odd = torch.zeros(D, D, device=DEV, dtype=torch.int64)
    for bit in range(D.bit_length()):
        odd ^= ((i[:, None] & i) >> bit) & 1
    return (1 - 2 * odd).double() / math.sqrt(D)


def _rows(cache, layer, s, name):
    """What the pages of a sequence hold, float64 [H, tokens, D], Hadamard-rotated."""
    pool = getattr(cache, name)[layer]
    if cache.k_bits == 8:
        val = ops.dequantize_q8(pool, getattr(cache, name + "_scale")[layer]).double()
    else:
        val = ops.dequantize(pool, cache.k_bits if name == "k" else 4).double()
    pages = torch.tensor(cache.pages.table[s, : cache.pages.n_pages[s]], device=DEV).long()
    return val[pages].transpose(0, 1).flatten(1, 2)


def _attend(q, k, v, sees):
    """q [Hq, n, D] over rows [H, T, D]; sees [n, T]."""
    had = _hadamard()
    x = (q.double() @ had).unflatten(0, (H, GRP))
    s = (x @ k[:, None].transpose(-1, -2)) / math.sqrt(D)
    p = torch.softmax(s.masked_fill(~sees, -math.inf), -1)
    return (p @ v[:, None] @ had).flatten(0, 1), s.flatten(0, 1)


def _make(k_bits, layers=2, **kw):
    cache = PagedKVCache(layers, H, D, num_pages=40, page_size=16, max_seqs=3, k_bits=k_bits, **kw)
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    return cache, rope, torch.Generator(device=DEV).manual_seed(k_bits)


def _step(cache, rope, g, step, observe=0, given=None, **kw):
    """One step of all layers with random (or given) inputs; returns the rotated queries and outputs of each layer."""
    out = []
    n = step.n_new
    for layer in range(cache.n_layers):
        k, v, q = given[layer] if given else (torch.randn(len(step.seqs), h, n, D, device=DEV, generator=g).bfloat16()
                                              for h in (H, H, H * GRP))
        qr = cache.append(step, layer, k, v, rope=rope, q=q)
        qa = qr if cache.k_bits == 8 else qr[:, :, -1].contiguous()
        out.append((qr, cache.attention(step, layer, qa, observe=observe, **kw), (k, v, q)))
    return out


def _near(got, want, tol=2e-3):
    assert float((got.double() - want).norm() / want.norm()) < tol


PARENTS = [-1, 0, 0, 1, 2, 2, 5, 3, -1]


@pytest.mark.parametrize("device_tree", [False, True])
def test_tree_steps(device_tree):
    cache, rope, g = _make(8)
    a, b = cache.add_sequence(), cache.add_sequence()
    step = cache.batch([a, b], [37, 20])
    _step(cache, rope, g, step)
    cache.commit(step)
    parents = torch.tensor(PARENTS, dtype=torch.int32, device=DEV) if device_tree else PARENTS
    n = len(PARENTS)
    step = cache.batch([a, b], n, tree=parents)
    assert step.positions.tolist() == [[s + d for d in (0, 1, 1, 2, 2, 2, 3, 3, 0)] for s in (37, 20)]
    seen = torch.eye(n, dtype=torch.bool)
    for i, p in enumerate(PARENTS):
        if p >= 0:
            seen[i] |= seen[p]
    got = _step(cache, rope, g, step, return_lse=True)
    for layer, (q, (out, lse), _) in enumerate(got):
        for i, s in enumerate((a, b)):
            past = cache.seq_len(s)
            k, v = (_rows(cache, layer, s, t)[:, : past + n] for t in "kv")
            sees = torch.cat((torch.ones(n, past, dtype=torch.bool), seen), 1).to(DEV)
            want, score = _attend(q[i], k, v, sees)
            _near(out[i], want)
            assert float((lse[i].double() - score.masked_fill(~sees, -math.inf).logsumexp(-1)).abs().max()) < 1e-2
    with pytest.raises(ValueError):
        cache.commit(step)                    # accept() commits a tree's step
    with pytest.raises(ValueError):
        cache.accept(step, [[0, 2, 5]])       # a path for each sequence
    for bad in ([0, 2, 1], [0, 9], [-1]) + (() if device_tree else ([0, 3], [1],)):
        with pytest.raises(ValueError):
            cache.accept(step, [bad, []])
    paths = [[0, 2, 5, 6], [8]]
    before = [[_rows(cache, layer, s, t) for t in "kv"] for layer in range(2) for s in (a, b)]
    kept = cache.accept(step, paths)
    assert (cache.seq_len(a), cache.seq_len(b)) == (41, 21) and kept.counts == [4, 1]
    # the rows of the path behind the cached ones, to half a step of 8 bits (twice: their blocks' scales may have grown)
    for layer in range(2):
        for i, (s, past) in enumerate(((a, 37), (b, 20))):
            for t in range(2):
                held = before[2 * layer + i][t]
                want = torch.cat((held[:, :past], held[:, [past + x for x in paths[i]]]), 1)
                now = _rows(cache, layer, s, "kv"[t])[:, : cache.seq_len(s)]
                step_of = (cache.k_scale, cache.v_scale)[t][layer].max().double()
                assert bool(((now - want).abs() <= step_of * 0.51).all())
    # steps go on: a chain of tokens behind the accepted path
    with pytest.raises(ValueError):
        cache.accept(step, paths)             # the sequences have changed
    step = cache.batch([a, b], 3)
    for layer, (q, out, _) in enumerate(_step(cache, rope, g, step)):
        for i, s in enumerate((a, b)):
            T = cache.seq_len(s) + 3
            k, v = (_rows(cache, layer, s, t)[:, :T] for t in "kv")
            sees = torch.arange(T, device=DEV) <= T - 3 + torch.arange(3, device=DEV)[:, None]
            _near(out[i], _attend(q[i], k, v, sees)[0])
    cache.commit(step)


def test_accepted_paths_are_a_chain():
    """A tree's accepted path leaves what the same tokens leave when they come as a chain: positions and order."""
    one, rope, g = _make(8, layers=1)
    two, _, _ = _make(8, layers=1)
    seqs = [one.add_sequence(), one.add_sequence()]
    assert seqs == [two.add_sequence(), two.add_sequence()]
    n, path = len(PARENTS), [0, 2, 5, 6]
    step = one.batch(seqs, n, tree=[PARENTS, PARENTS])
    (_, _, (k, v, q)), = _step(one, rope, g, step)
    one.accept(step, [path, path])
    chain = two.batch(seqs, len(path))
    _step(two, rope, g, chain, given=[(k[:, :, path], v[:, :, path], q[:, :, path])])
    two.commit(chain)
    for s in seqs:
        for t in "kv":
            x, y = (_rows(c, 0, s, t)[:, :4] for c in (one, two))
            scale = max(float(getattr(c, t + "_scale")[0].max()) for c in (one, two))
            assert bool(((x - y).abs() <= 1.51 * scale).all())     # half a step in each cache, and half of another when moved


@pytest.mark.parametrize("k_bits", [8, 3, 4, 2])
def test_eviction(k_bits):
    cache, rope, g = _make(k_bits, track_weights=True)
    a, b, c = (cache.add_sequence() for _ in range(3))
    lens = {a: 0, b: 0, c: 0}

    def run(seqs, n, observe=1, decay=1.0):
        step = cache.batch(seqs, n)
        got = _step(cache, rope, g, step, observe=observe, decay=decay)
        cache.commit(step)
        for s, m in zip(seqs, step.counts or [step.n_new] * len(seqs)):
            lens[s] += m
        return step, got

    run([a, b, c], [60, 33, 9] if k_bits == 8 else 60, observe=16 if k_bits == 8 else 1)
    for _ in range(5):
        run([a, b, c], 1, decay=0.9)
    before = {(layer, s, t): _rows(cache, layer, s, t) for layer in range(2) for s in (a, b, c) for t in "kv"}
    sums = {}
    for layer in range(2):
        for s in (a, b, c):
            pages = torch.tensor(cache.pages.table[s, : cache.pages.n_pages[s]], device=DEV).long()
            sums[layer, s] = cache.weights[layer][pages].transpose(0, 1).flatten(1)
            w = sums[layer, s][:, : lens[s]]
            # every query row's weights add up to one: the earlier rows' times decay for each later step
            if k_bits != 8:
                total = GRP * sum(0.9 ** (5 - i) for i in range(6))
                assert float((w.double().sum(-1) - total).abs().max()) < 0.02 * total
    free = cache.pages.free_pages
    keep = [20, lens[b], 7]
    cache.evict([a, b, c], keep, sinks=2, recent=4)
    left = [min(n, lens[s]) for s, n in zip((a, b, c), keep)]
    assert [cache.seq_len(s) for s in (a, b, c)] == left
    assert cache.pages.free_pages == free + sum(-(-lens[s] // 16) - (-(-n // 16)) for s, n in zip((a, b, c), left))
    for layer in range(2):
        for s, n in zip((a, b, c), left):
            w = sums[layer, s][:, : lens[s]].clone()
            if n < lens[s]:
                w[:, :2] = w[:, lens[s] - 4:] = math.inf
            kept = w.sort(dim=1, descending=True, stable=True).indices[:, :n].sort(dim=1).values
            for t in "kv":
                want = before[layer, s, t].gather(1, kept[..., None].expand(-1, -1, D))
                now = _rows(cache, layer, s, t)[:, :n]
                if k_bits == 8:
                    tol = 0.51 * float(getattr(cache, t + "_scale")[layer].max())
                    assert bool(((now - want).abs() <= tol).all())
                else:
                    assert torch.equal(now, want)
    # the next steps see the kept tokens, their own positions behind all tokens that there were
    for n in ([1, 3] if k_bits == 8 else [1, 1]):
        first = [lens[s] for s in (a, b, c)]
        step, got = run([a, b, c], n)
        if first[0] > left[0]:
            assert step.positions[:, 0].tolist() == first
        for layer, (q, out, (k, v, q0)) in enumerate(got):
            where = torch.tensor(first, dtype=torch.int32, device=DEV)[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)
            assert torch.equal(q, ops.rotary(q0, where.contiguous(), rope))
            for i, s in enumerate((a, b, c)):
                T = cache.seq_len(s)
                kk, vv = (_rows(cache, layer, s, t)[:, :T] for t in "kv")
                sees = torch.arange(T, device=DEV) <= T - n + torch.arange(n, device=DEV)[:, None]
                want = _attend(q[i], kk, vv, sees)[0]
                _near(out[i] if k_bits == 8 else out[i][:, None], want, 3e-3)
    cache.evict([a], 1 << 20)                  # more than there are: nothing happens
    cache.free_sequence(a)
    again = cache.add_sequence()
    lens[again] = 0
    step, _ = run([again], 5)
    assert step.positions is None
    # a page's new owner does not count what the old one had
    pages = torch.tensor(cache.pages.table[again, :1], device=DEV).long()
    assert bool((cache.weights[0][pages][:, :, 5:] == 0).all())


def test_observed_after_acceptance():
    """The accepted rows' weights, counted after the move with the log-sum-exps that the tree's attention left."""
    cache, rope, g = _make(8, layers=1, track_weights=True)
    a = cache.add_sequence()
    step = cache.batch([a], 30)
    _step(cache, rope, g, step, observe=30)
    cache.commit(step)
    step = cache.batch([a], len(PARENTS), tree=PARENTS)
    with pytest.raises(ValueError):
        _step(cache, rope, g, step, observe=1)
    (q, (_, lse), _), = _step(cache, rope, g, step, return_lse=True)
    path = [0, 1, 3]
    start = cache.weights[0].clone()
    kept = cache.accept(step, [path])
    cache.observe(kept, 0, q[:, :, path], lse[:, :, path].contiguous(), decay=0.5)
    k = _rows(cache, 0, a, "k")[:, :33]
    had = _hadamard()
    s = (q[0][:, path].double() @ had).unflatten(0, (H, GRP)) @ k[:, None].transpose(-1, -2) / math.sqrt(D)
    sees = torch.arange(33, device=DEV) <= 30 + torch.arange(3, device=DEV)[:, None]
    p = torch.where(sees, torch.exp(s - lse[0][:, path].double().unflatten(0, (H, GRP))[..., None]), 0.0).sum((1, 2))
    pages = torch.tensor(cache.pages.table[a, :3], device=DEV).long()
    had_before = start[pages].transpose(0, 1).flatten(1)[:, :33].double()
    had_before[:, 30:] = 0
    now = cache.weights[0][pages].transpose(0, 1).flatten(1)[:, :33].double()
    _near(now, 0.5 * had_before + p, 1e-5)


@pytest.mark.parametrize("k_bits", [8, 3])
def test_rejected_drafts_leave_no_weights(k_bits):
    cache, rope, g = _make(k_bits, track_weights=True)
    s = cache.add_sequence()

    def held():
        pages = torch.tensor(cache.pages.table[s, : cache.pages.n_pages[s]], device=DEV).long()
        return torch.stack([w[pages].transpose(0, 1).flatten(1) for w in cache.weights])

    step = cache.batch([s], 30)
    _step(cache, rope, g, step) if k_bits == 8 else None
    if k_bits != 8:   # TurboQuant keys: one query a sequence
        for layer in range(2):
            k, v = (torch.randn(1, H, 30, D, device=DEV, generator=g).bfloat16() for _ in range(2))
            cache.append(step, layer, k, v)
    cache.commit(step)
    drafted = cache.batch([s], 6)
    for layer in range(2):
        k, v, q = (torch.randn(1, h, 6, D, device=DEV, generator=g).bfloat16() for h in (H, H, H * GRP))
        cache.append(drafted, layer, k, v)
        cache.attention(drafted, layer, q if k_bits == 8 else q[:, :, -1], observe=6)
    assert bool((held()[..., :36] > 0).all())
    cache.commit(cache.batch([s], 3))   # slots 33 .. 35 held rejected tokens
    assert bool((held()[..., :33] > 0).all()) and bool((held()[..., 33:] == 0).all())
    cache.commit(cache.batch([s], 20))   # not observed
    assert bool((held()[..., :33] > 0).all()) and bool((held()[..., 33:] == 0).all())


def test_refusals():
    plain = PagedKVCache(1, H, D, num_pages=8, page_size=16, max_seqs=2, k_bits=8)
    s = plain.add_sequence()
    step = plain.batch([s], 2)
    q = torch.zeros(1, H * GRP, 2, D, device=DEV, dtype=torch.bfloat16)
    for call in (lambda: plain.evict([s], 1), lambda: plain.attention(step, 0, q, observe=1), lambda: plain.accept(step, [[0]]),
                 lambda: plain.batch([s], 3, tree=[-1, 0]), lambda: plain.batch([s], 2, tree=[0, 0]), lambda: plain.batch([s], 2, tree=[-2, 0]),
                 lambda: plain.batch([s], 2, tree=[[-1, 0], [-1, 0]])):
        with pytest.raises(ValueError):
            call()
    # a step made before an eviction, and one of a sequence that has gone
    kept = PagedKVCache(1, H, D, num_pages=8, page_size=16, max_seqs=2, k_bits=8, track_weights=True)
    s = kept.add_sequence()
    kept.commit(kept.batch([s], 20))
    old, tree = kept.batch([s], 1), kept.batch([s], 2, tree=[-1, 0])
    kept.evict([s], 10)
    for call in (lambda: kept.commit(old), lambda: kept.accept(tree, [[0]])):
        with pytest.raises(ValueError):
            call()
    tree = kept.batch([s], 2, tree=[-1, 0])
    kept.free_sequence(s)
    with pytest.raises(ValueError):
        kept.accept(tree, [[0]])
    tq = PagedKVCache(1, H, D, num_pages=8, page_size=16, max_seqs=2, k_bits=3)
    with pytest.raises(ValueError):
        tq.batch([tq.add_sequence()], 2, tree=[-1, 0])
    assert attention.last_status() == 0
