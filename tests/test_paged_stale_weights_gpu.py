"""Observed weights of PagedKVCache when drafted tokens are dropped and others take their slots, and beside evictions of other sequences:
a token's weights are those that it was given itself."""
import pytest
import torch

from leankv_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, GRP, D, LAYERS = 2, 4, 128, 3


def _cache(bits, **kw):
    cache = PagedKVCache(LAYERS, H, D, num_pages=24, page_size=16, max_seqs=3, k_bits=bits, track_weights=True, **kw)
    return cache, torch.Generator(device=DEV).manual_seed(bits)


def _held(cache, s):
    """The weights of a sequence's slots [layers, H, slots]."""
    pages = torch.tensor(cache.pages.table[s, : cache.pages.n_pages[s]], device=DEV).long()
    return torch.stack([w[pages].transpose(0, 1).flatten(1) for w in cache.weights])


def _run(cache, g, step, observed=()):
    """Appends the step's rows in every layer, and attends with the last query observed in some."""
    n, B = step.n_new, len(step.seqs)
    for layer in range(LAYERS):
        k, v, q = (torch.randn(B, h, n, D, device=DEV, generator=g).bfloat16() for h in (H, H, H * GRP))
        cache.append(step, layer, k, v)
        cache.attention(step, layer, q if cache.k_bits == 8 else q[:, :, -1], observe=n if layer in observed else 0)


@pytest.mark.parametrize("bits", [8, 3])
@pytest.mark.parametrize("layers", [(), (0,), (2, 1)])
def test_tokens_in_the_slots_of_dropped_drafts(bits, layers):
    cache, g = _cache(bits)
    s = cache.add_sequence()
    step = cache.batch([s], 30)
    _run(cache, g, step, range(LAYERS))
    cache.commit(step)
    _run(cache, g, cache.batch([s], 9), range(LAYERS))    # drafted, observed, and dropped
    assert bool((_held(cache, s)[..., 30:39] > 0).all())
    step = cache.batch([s], 4)
    _run(cache, g, step, layers)
    cache.commit(step)
    held = _held(cache, s)
    for layer in range(LAYERS):
        assert bool((held[layer, :, :30] > 0).all()) and bool((held[layer, :, 34:] == 0).all())
        assert bool((held[layer, :, 30:34] > 0).all() if layer in layers else (held[layer, :, 30:34] == 0).all())


@pytest.mark.parametrize("bits", [8, 3])
def test_a_prefix_of_drafts_behind_dropped_ones(bits):
    cache, g = _cache(bits)
    s = cache.add_sequence()
    _run(cache, g, cache.batch([s], 9), range(LAYERS))    # dropped
    _run(cache, g, cache.batch([s], 7), (1,))             # of these three stay
    cache.commit(cache.batch([s], 3))
    held = _held(cache, s)
    assert bool((held[1, :, :3] > 0).all()) and bool((held[1, :, 3:] == 0).all())
    assert bool((held[0] == 0).all()) and bool((held[2] == 0).all())


def test_accepted_nodes_in_the_slots_of_dropped_drafts():
    cache, g = _cache(8)
    s = cache.add_sequence()
    step = cache.batch([s], 20)
    _run(cache, g, step, range(LAYERS))
    cache.commit(step)
    _run(cache, g, cache.batch([s], 6), range(LAYERS))
    tree = cache.batch([s], 5, tree=[-1, 0, 0, 1, 2])
    _run(cache, g, tree)
    kept = cache.accept(tree, [[0, 2, 4]])
    held = _held(cache, s)
    assert bool((held[..., :20] > 0).all()) and bool((held[..., 20:] == 0).all())
    q = torch.randn(1, H * GRP, 3, D, device=DEV, generator=g).bfloat16()
    cache.observe(kept, 1, q, torch.full((1, H * GRP, 3), 4.0, device=DEV))
    assert bool((_held(cache, s)[1, :, 20:23] > 0).all())


def test_a_step_written_twice():
    cache, g = _cache(8)
    s = cache.add_sequence()
    step = cache.batch([s], 5)
    _run(cache, g, step, range(LAYERS))
    _run(cache, g, step)      # other rows, not observed
    cache.commit(step)
    assert bool((_held(cache, s) == 0).all())


@pytest.mark.parametrize("bits", [8, 3])
def test_a_step_under_way_beside_an_eviction(bits):
    """A sequence that keeps all its tokens keeps the pages and the weights of a step that is still to be committed."""
    cache, g = _cache(bits)
    a, b = cache.add_sequence(), cache.add_sequence()
    step = cache.batch([a, b], 30)
    _run(cache, g, step, range(LAYERS))
    cache.commit(step)
    step = cache.batch([b], 5)            # its last three slots are on a page that no token has yet
    _run(cache, g, step, range(LAYERS))
    before, held = _held(cache, b), list(cache.pages.table[b])
    cache.evict([a, b], [12, 100], sinks=1, recent=2)
    assert (cache.seq_len(a), cache.seq_len(b)) == (12, 30) and list(cache.pages.table[b]) == held
    cache.commit(step)
    assert cache.seq_len(b) == 35 and torch.equal(_held(cache, b), before) and bool((before[..., :35] > 0).all())
