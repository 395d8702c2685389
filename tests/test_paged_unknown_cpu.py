"""Sequences that a cache does not have: refused alike with and without weights (no GPU)."""
import pytest

from leankv_b200.paged import PagedKVCache


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("unknown", [1, 2, -1, 1 << 40])
def test_unknown_sequences(track, unknown):
    cache = PagedKVCache(1, 1, 128, num_pages=4, page_size=16, max_seqs=2, k_bits=8, device="cpu", track_weights=track)
    s = cache.add_sequence()
    for call in (lambda: cache.batch([s, unknown], 1), lambda: cache.batch([unknown], 2, tree=[-1, 0]), lambda: cache.free_sequence(unknown)):
        with pytest.raises(ValueError):
            call()
    if track:
        with pytest.raises(ValueError):
            cache.evict([unknown], 1)
    assert cache.pages.free_pages == 4
