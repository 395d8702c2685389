"""Calls of tensors on a device that is not the current one (no GPU: the device, its guard and the library are stand-ins):
the work memory is sized on the tensors' device, as the launch plans it, since the plan depends on its SMs."""
import contextlib

import torch

from leankv_b200 import attention, ops


class _Library:
    """Plans by the current device; a launch refuses work memory of another device's plan, as the library does."""

    def __init__(self, current):
        self.current, self.seen = current, []

    def _size(self):
        return {0: 1 << 10, 1: 1 << 12}[self.current[0]]

    def tq_attention_q8_workspace_size(self, args, pages):
        self.seen.append(("size", self.current[0]))
        return self._size()

    def tq_attention_q8_paged_cuda(self, args, pages, stream):
        self.seen.append(("launch", self.current[0], stream))
        return 0 if attention._ATTN_Q8.unpack(args)[-1] >= self._size() else 1

    @staticmethod
    def tq_last_error_string():
        return b"workspace too small"


def test_work_memory_is_sized_on_the_tensors_device(monkeypatch):
    current = [0]
    lib = _Library(current)

    @contextlib.contextmanager
    def guard(device):
        before, current[0] = current[0], device
        yield
        current[0] = before

    monkeypatch.setattr(attention.L, "load", lambda: lib)
    monkeypatch.setattr(attention, "_device_of", lambda *ts: 1)
    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 100 + device)
    monkeypatch.setattr(torch.cuda, "device", guard)
    q = torch.zeros(1, 2, 1, 128)
    pool, scale = torch.zeros(4, 1, 16, 128, dtype=torch.int8), torch.zeros(4, 1, 1)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    attention.attention_q8_paged(q, pool, pool, scale, scale, table, lens)
    assert lib.seen == [("size", 1), ("launch", 1, 101)] and current == [0]
    # on the current device: no guard
    lib.seen.clear()
    monkeypatch.setattr(attention, "_device_of", lambda *ts: 0)
    monkeypatch.setattr(torch.cuda, "device", None)
    attention.attention_q8_paged(q, pool, pool, scale, scale, table, lens)
    assert lib.seen == [("size", 0), ("launch", 0, 100)]
