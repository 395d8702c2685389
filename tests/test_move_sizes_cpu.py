"""Work memory of calls that move rows, whatever calls of the same sizes came before (no GPU: sizes are the library's, launches are not made)."""
import pytest
import torch

from leankv_b200 import _lib as L
from leankv_b200 import ops

H, D, P, PER, ROWS = 2, 128, 16, 20, 130


class _Library:
    def __init__(self, real):
        self.real, self.given = real, []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def tq_kv_move_paged_cuda(self, args, pages, stream):
        self.given.append((ops._MOVE.unpack(args)[-1], self.real.tq_kv_move_workspace_size(args, pages)))
        return 0


@pytest.fixture
def library(monkeypatch):
    lib = _Library(L.load())
    monkeypatch.setattr(L, "load", lambda: lib)
    monkeypatch.setattr(ops, "_device_of", lambda *ts: 0)
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_work_sizes", {})
    return lib


def _move(to=None):
    pool, scale = torch.zeros(2 * PER, H, P, D, dtype=torch.int8), torch.zeros(2 * PER, H, P // 16)
    table = torch.arange(PER, dtype=torch.int32).view(1, PER)
    to_table = {None: None, "same": table, "other": table + PER}[to]
    ops.kv_move_paged(pool, pool, table, torch.zeros(1, H, ROWS, dtype=torch.int32), k_scale=scale, v_scale=scale, to_table=to_table)


@pytest.mark.parametrize("order", [("other", "same"), ("same", "other"), ("other", None, "same", "other"), (None, "other")])
def test_work_memory_does_not_depend_on_the_order_of_calls(library, order):
    for to in order:
        _move(to)
    assert all(given == needed for given, needed in library.given)
    assert [needed > 0 for _, needed in library.given] == [to != "other" for to in order]


def test_a_destination_without_pages_is_refused(library):
    pool, scale = torch.zeros(4, H, P, D, dtype=torch.int8), torch.zeros(4, H, P // 16)
    with pytest.raises(ValueError):
        ops.kv_move_paged(pool, pool, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, H, 3, dtype=torch.int32), k_scale=scale,
                          v_scale=scale, to_table=torch.zeros(1, 0, dtype=torch.int32))
    assert not library.given
