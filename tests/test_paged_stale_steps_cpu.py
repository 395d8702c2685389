"""Steps of PagedKVCache that outlive pages of their sequences: refused by whatever would read or write through them (no GPU)."""
import pytest
import torch

from leankv_b200 import attention, ops
from leankv_b200.paged import PagedKVCache

H, D = 1, 128


@pytest.fixture
def calls(monkeypatch):
    """The device calls that the cache makes, by name, in place of kernels."""
    made = []

    def fake(name, result=None):
        def call(*args, **kw):
            made.append(name)
            return result
        return call
    for module, name in ((ops, "kv_append_paged"), (ops, "kv_append_rotary_paged"), (ops, "select_tokens"), (ops, "kv_move_paged"),
                         (attention, "attention_q8_paged"), (attention, "attention_weights_paged"), (attention, "decode_attention_paged")):
        monkeypatch.setattr(module, name, fake(name, (None, None)))
    monkeypatch.setattr(ops, "draft_tree", lambda parents: ops.DraftTree(torch.zeros(1, parents.shape[-1], 1, dtype=torch.int32),
                                                                         torch.zeros(1, parents.shape[-1], dtype=torch.int32)))
    return made


def _cache(bits=8):
    return PagedKVCache(1, H, D, num_pages=6, page_size=16, max_seqs=3, k_bits=bits, device="cpu", track_weights=True)


def _uses(cache, step):
    n = step.n_new
    k = torch.zeros(len(step.seqs), H, n, D)
    lse = torch.zeros(len(step.seqs), H, n)
    yield "append", lambda: cache.append(step, 0, k, k)
    yield "attention", lambda: cache.attention(step, 0, k)
    yield "attention that observes", lambda: cache.attention(step, 0, k, observe=1)
    yield "observe", lambda: cache.observe(step, 0, k, lse)
    yield "commit", lambda: cache.commit(step)


def _refused(cache, step, calls):
    for name, use in _uses(cache, step):
        calls.clear()
        with pytest.raises(ValueError, match="since the step was made"):
            use()
        assert not calls, name


def test_after_an_eviction(calls):
    cache = _cache()
    a, b = cache.add_sequence(), cache.add_sequence()
    cache.commit(cache.batch([a, b], 40))
    old, other = cache.batch([a, b], 1), cache.batch([b], 1)
    cache.evict([a], 10)
    taken = cache.batch([b], 20)                # takes a page that a has given back
    assert set(taken.table[0].tolist()) & set(old.table[0].tolist()) - {-1}
    _refused(cache, old, calls)
    for _, use in _uses(cache, other):          # steps of other sequences go on
        use()


def test_of_a_sequence_that_was_freed_and_another_in_its_place(calls):
    cache = _cache()
    a = cache.add_sequence()
    old = cache.batch([a], 20)
    cache.free_sequence(a)
    _refused(cache, old, calls)
    assert cache.add_sequence() == a
    _refused(cache, old, calls)
    new = cache.batch([a], 20)
    for _, use in _uses(cache, new):
        use()


def test_accepted_steps_and_trees(calls):
    cache = _cache()
    a = cache.add_sequence()
    cache.commit(cache.batch([a], 30))
    tree = cache.batch([a], 3, tree=[-1, 0, 0])
    kept = cache.accept(tree, [[0, 1]])
    pending = cache.batch([a], 2, tree=[-1, 0])
    cache.evict([a], 8)
    calls.clear()
    q = torch.zeros(1, H, 2, D)
    with pytest.raises(ValueError, match="since the step was made"):
        cache.observe(kept, 0, q, torch.zeros(1, H, 2))
    with pytest.raises(ValueError, match="since the step was made"):
        cache.accept(pending, [[0]])
    assert not calls and cache.seq_len(a) == 8


def test_an_eviction_that_drops_nothing(calls):
    cache = _cache()
    a = cache.add_sequence()
    cache.commit(cache.batch([a], 30))
    step = cache.batch([a], 1)
    cache.evict([a], 30)
    for _, use in _uses(cache, step):
        use()
