"""PagedKVCache steps with the position rotation on the way and with 8-bit pages: sequences join, leave and bring
different numbers of tokens; at every step and layer the cache's pools and outputs equal the single calls', and
8-bit attention stays near attention over the unquantized rows."""
import math

import pytest
import torch

from leankv_b200 import attention, ops
from leankv_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rows(B, n, hq, hk, D, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(B, n, hq + 2 * hk, D, device=DEV, generator=g).bfloat16()
    return tuple(t.transpose(1, 2) for t in x.split([hq, hk, hk], dim=2))


@pytest.mark.parametrize("k_bits,k_opt", [(3, 0), (4, 0), (2, 0), (3, 2)])
def test_rotary_steps_equal_rotation_then_append(k_bits, k_opt):
    D, hk, grp = 128, 2, 4
    make = lambda: PagedKVCache(1, hk, D, num_pages=40, page_size=16, max_seqs=4, k_bits=k_bits, k_opt_passes=k_opt)   # noqa: E731
    one, two = make(), make()
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    seqs = [one.add_sequence(), one.add_sequence()]
    assert seqs == [two.add_sequence(), two.add_sequence()]
    for seed, n in enumerate([37, 1, 5, 1]):
        q, k, v = _rows(2, n, hk * grp, hk, D, seed)
        a, b = one.batch(seqs, n), two.batch(seqs, n)
        where = (a.pos[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)).contiguous()
        got = one.append(a, 0, k, v, rope=rope, q=q)
        want, turned = ops.rotary(q, where, rope), ops.rotary(k.float(), where, rope)
        assert two.append(b, 0, turned, v) is None
        assert torch.equal(got, want) and torch.equal(one.k[0], two.k[0]) and torch.equal(one.v[0], two.v[0])
        last = got[:, :, -1].contiguous()
        assert torch.equal(one.attention(a, 0, last), two.attention(b, 0, last))
        one.commit(a)
        two.commit(b)


@pytest.mark.parametrize("D,page_size", [(128, 16), (256, 64)])
def test_q8_cache_steps(D, page_size):
    layers, hk, grp = 2, 2, 4
    cache = PagedKVCache(layers, hk, D, num_pages=80, page_size=page_size, max_seqs=4, max_pages_per_seq=40, k_bits=8)
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    held = {}
    plan = [("join", 2), ("step", [50, 3]), ("step", 1), ("join", 1), ("step", [1, 0, 150]), ("step", 4), ("leave", 0),
            ("step", [1, 1]), ("join", 1), ("step", [2, 1, 60]), ("step", 1)]
    seqs = []
    for op, n in plan:
        if op == "join":
            for _ in range(n):
                s = cache.add_sequence()
                seqs.append(s)
                held[s] = [[] for _ in range(layers)]
            continue
        if op == "leave":
            cache.free_sequence(seqs.pop(n))
            continue
        step = cache.batch(seqs, n)
        B, rows = len(seqs), step.n_new
        counts = n if isinstance(n, list) else [n] * B
        assert rows == max(counts) and step.kv_len.tolist() == [cache.seq_len(s) + c for s, c in zip(seqs, counts)]
        for layer in range(layers):
            q, k, v = _rows(B, rows, hk * grp, hk, D, 100 * len(held) + 7 * rows + layer)
            where = (step.pos[:, None] + torch.arange(rows, dtype=torch.int32, device=DEV)).contiguous()
            kr = ops.rotary(k.float(), where, rope)
            qr = cache.append(step, layer, k, v, rope=rope, q=q)
            assert torch.equal(qr, ops.rotary(q, where, rope))
            out = cache.attention(step, layer, qr)
            single = attention.attention_q8_paged(qr, cache.k[layer], cache.v[layer], cache.k_scale[layer], cache.v_scale[layer],
                                                  step.table, step.kv_len, q_len=step.new_len, max_kv_len=step.max_kv_len)
            assert torch.equal(out, single)
            for b, s in enumerate(seqs):
                c = counts[b]
                held[s][layer].append((kr[b, :, :c], v[b, :, :c].float()))
                assert bool((out[b, :, c:] == 0).all())
                if not c:
                    continue
                K, V = (torch.cat(t, 1).double().repeat_interleave(grp, 0) for t in zip(*held[s][layer]))
                L = K.shape[1]
                w = qr[b, :, :c].double() @ K.transpose(1, 2) / math.sqrt(D)
                hide = torch.arange(L, device=DEV) > (L - c + torch.arange(c, device=DEV))[:, None]
                want = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ V
                # codes are steps of a block's largest of 16 D rotated elements (about 4.3 deviations) / 127: errors of
                # 0.01 deviations of values and, over the D terms of a score / sqrt(D), of scores
                assert float((out[b, :, :c].double() - want).norm() / want.norm()) < 0.03
        cache.commit(step)
    # the second sequence to join, the one that joined later, the last
    assert [cache.seq_len(s) for s in seqs] == [3 + 1 + 0 + 4 + 1 + 2 + 1, 150 + 4 + 1 + 1 + 1, 60 + 1]
    assert cache.memory_summary()["pages_used"] == sum(-(-cache.seq_len(s) // page_size) for s in seqs)


def test_q8_cache_refusals():
    cache = PagedKVCache(1, 2, 128, num_pages=8, k_bits=8)
    s = cache.add_sequence()
    with pytest.raises(ValueError):
        cache.batch([s], [1, 2])
    with pytest.raises(ValueError):
        cache.batch([s], [-1])
    step = cache.batch([s], 4)
    q, k, v = _rows(1, 4, 4, 2, 128, 1)
    with pytest.raises(ValueError):
        cache.append(step, 0, k, v, q=q)
    with pytest.raises(ValueError):
        cache.append(step, 0, k[:, :, :2], v[:, :, :2])
    cache.append(step, 0, k, v)
    with pytest.raises(ValueError):
        cache.attention(step, 0, q[:, :, :2])
    with pytest.raises(ValueError):
        PagedKVCache(1, 2, 128, num_pages=8, k_bits=5)
    opt = PagedKVCache(1, 2, 128, num_pages=8, k_bits=3, k_opt_passes=2)
    a, b = opt.add_sequence(), opt.add_sequence()
    step = opt.batch([a, b], [1, 2])
    q, k, v = _rows(2, 2, 4, 2, 128, 1)
    with pytest.raises(ValueError):
        opt.append(step, 0, k, v)


def test_q8_one_row_each_and_padding():
    """A step of one row or none for each sequence: a row of padding gives zeros in either shape of q; one row out of a
    step of several is each sequence's last."""
    D, hk, grp = 128, 2, 4
    cache = PagedKVCache(1, hk, D, num_pages=16, page_size=16, max_seqs=2, k_bits=8)
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    seqs = [cache.add_sequence(), cache.add_sequence()]
    for seed, counts in enumerate([[20, 33], [1, 0]]):
        step = cache.batch(seqs, counts)
        q, k, v = _rows(2, step.n_new, hk * grp, hk, D, seed)
        q = cache.append(step, 0, k, v, rope=rope, q=q)
        every = cache.attention(step, 0, q)
        if step.n_new == 1:
            one = cache.attention(step, 0, q[:, :, 0])
            assert torch.equal(one, every[:, :, 0])
            assert not one[1].any() and one[0].any()
        else:
            last = torch.stack([q[b, :, n - 1] for b, n in enumerate(counts)])
            one = cache.attention(step, 0, last)
            for b, n in enumerate(counts):   # the same scores in other sums: both are within 2^-8 of the true values' norm
                x, y = one[b].double(), every[b, :, n - 1].double()
                assert (x - y).norm() <= 2 * 2.0 ** -8 * y.norm()
        cache.commit(step)
