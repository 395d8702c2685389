"""Page bookkeeping of steps whose sequences bring different numbers of tokens (no GPU)."""
import pytest

from leankv_b200.paged import PageTable


def test_reserve_and_commit_with_a_count_each():
    pt = PageTable(num_pages=10, page_size=16, max_seqs=3, max_pages_per_seq=5)
    a, b, c = (pt.add_sequence() for _ in range(3))
    pt.reserve([a, b, c], [17, 0, 16])
    assert [int(pt.n_pages[s]) for s in (a, b, c)] == [2, 0, 1] and pt.free_pages == 7
    pt.commit([a, b, c], [17, 0, 16])
    assert [int(pt.lens[s]) for s in (a, b, c)] == [17, 0, 16]
    pt.reserve([a, b, c], 1)
    assert [int(pt.n_pages[s]) for s in (a, b, c)] == [2, 1, 2]
    with pytest.raises(ValueError):
        pt.commit([a, b], [1, 17])       # b holds one page
    with pytest.raises(ValueError):
        pt.reserve([a, b], [1])
    with pytest.raises(ValueError):
        pt.reserve([a, b], [1, -1])
    with pytest.raises(MemoryError):
        pt.reserve([a, b], [48, 64])     # 3 + 3 pages needed, 5 free
    assert pt.free_pages == 5
