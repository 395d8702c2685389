"""Rotary and 8-bit page entry points without a GPU: statuses of refused arguments (set before any device
work), the helpers that build frequencies and axes, and the argument blocks' layouts."""
import ctypes as C
import subprocess

import pytest
import torch

from leankv_b200 import _lib as L
from leankv_b200 import ops


def _rope(**kw):
    base = dict(inv_freq=64, axis=None, positions=64, n_axes=1, rotary_dim=64, interleaved=0, inverse=0, scale=1.0)
    return ops._Rope(**{**base, **kw})


def _heads(**kw):
    base = dict(src=64, dst=64, heads=2, src_stride=(1024, 128, 256), dst_stride=(1024, 128, 256))
    return ops._HeadRows(**{**base, **kw})


@pytest.mark.parametrize("rope,dtype,batch,n,D,x,status", [
    (dict(rotary_dim=24), 1, 1, 1, 64, {}, 1), (dict(rotary_dim=128), 1, 1, 1, 64, {}, 1),
    (dict(inv_freq=None), 1, 1, 1, 64, {}, 1), (dict(positions=None), 1, 1, 1, 64, {}, 1),
    (dict(n_axes=0), 1, 1, 1, 64, {}, 1), (dict(scale=float("inf")), 1, 1, 1, 64, {}, 1),
    (dict(inv_freq=68), 1, 1, 1, 64, {}, 3), (dict(positions=66), 1, 1, 1, 64, {}, 3),
    ({}, 5, 1, 1, 64, {}, 1), ({}, 1, -1, 1, 64, {}, 1), ({}, 1, 1, -1, 64, {}, 1), ({}, 1, 1, 1 << 31, 64, {}, 1),
    ({}, 1, 1, 1, 68, {}, 2), ({}, 1, 1, 1, 520, {}, 2), ({}, 1, 1, 1, 64, dict(heads=0), 1),
    ({}, 1, 1, 1, 64, dict(src=None), 1), ({}, 1, 1, 1, 64, dict(src=72), 3),
    ({}, 1, 1, 1, 64, dict(src_stride=(1024, 128, 132), dst=128), 3),
    ({}, 1, 1, 1, 64, dict(src_stride=(1024, 128, 512)), 1),
    ({}, 1, 0, 1, 64, {}, 0), ({}, 1, 1, 0, 64, {}, 0)])
def test_rotary_statuses(rope, dtype, batch, n, D, x, status):
    lib = L.load()
    got = lib.tq_rotary_cuda(C.byref(_rope(**rope)), dtype, batch, n, D, C.byref(_heads(**x)), None, None)
    assert got == status
    assert status == 0 or lib.tq_last_error_string()


def _append(**kw):
    h = _heads(dst=None)
    base = dict(batch=1, n_kv_heads=2, head_dim=128, n_new=1, dtype=1, k=h, v=h, q=ops._HeadRows(), rope=_rope(rotary_dim=128, positions=None),
                k_pool=64, k_type=8, k_scale=64, v_pool=64, v_type=8, v_scale=64, pos=None, new_len=None, rotate=1, overflow=None)
    return ops._RotaryAppendArgs(**{**base, **kw})


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), 1), (dict(n_kv_heads=0), 1), (dict(head_dim=64), 2), (dict(k_type=3), 2), (dict(k_type=5), 2),
    (dict(v_type=4), 2), (dict(rope=_rope(rotary_dim=128, inverse=1)), 1),
    (dict(rope=_rope(rotary_dim=128, positions=None, n_axes=3)), 1),
    (dict(rope=ops._Rope(), q=_heads()), 1), (dict(k=_heads(heads=3)), 1), (dict(v=_heads(src=None)), 1),
    (dict(q=_heads(dst=None)), 1), (dict(k_scale=None), 1), (dict(v_pool=None), 1), (dict(k_pool=72), 3),
    (dict(v_scale=66), 3), (dict(pos=66), 3), (dict(q=_heads(heads=-1)), 1), (dict(n_new=0), 0), (dict(batch=0), 0)])
def test_append_statuses(change, status):
    from leankv_b200.attention import KVPages
    pages = KVPages(64, 4, 8, 16)
    assert L.load().tq_kv_append_rotary_paged_cuda(C.byref(_append(**change)), C.byref(pages), None) == status
    assert L.load().tq_kv_append_rotary_paged_cuda(C.byref(_append()), C.byref(KVPages(64, 4, 8, 24)), None) == 1
    assert L.load().tq_kv_append_rotary_paged_cuda(C.byref(_append()), None, None) == 1


@pytest.mark.parametrize("args,status", [
    ((64, 64, 64, 7, 1, 128), 1), ((64, 64, 64, 0, 1, 64), 2), ((64, 64, 64, 0, -1, 128), 1), ((None, 64, 64, 0, 1, 128), 1),
    ((72, 64, 64, 0, 1, 128), 3), ((64, 66, 64, 0, 1, 128), 3), ((None, None, None, 0, 0, 128), 0)])
def test_dequantize_q8_statuses(args, status):
    assert L.load().tq_dequantize_q8_cuda(*args, None) == status


def test_argument_blocks_match_the_header(tmp_path):
    src = tmp_path / "s.c"
    src.write_text('#include "leankv_tq.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){ printf("%zu %zu %zu %zu %zu\\n",'
                   ' sizeof(tq_rope), sizeof(tq_head_rows), sizeof(tq_rotary_append_args), offsetof(tq_rotary_append_args, rope),'
                   ' offsetof(tq_rotary_append_args, overflow)); return 0; }\n')
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", L.HEADER_DIR, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    A = ops._RotaryAppendArgs
    assert got == [C.sizeof(ops._Rope), C.sizeof(ops._HeadRows), C.sizeof(A), A.rope.offset, A.overflow.offset]


def test_frequencies_and_axes():
    f = ops.rotary_frequencies(8, theta=16.0, device="cpu")
    assert f.dtype == torch.float64 and f.tolist() == [1.0, 0.5, 0.25, 0.125]
    assert ops.rotary_axes((1, 2, 1), "cpu").tolist() == [0, 1, 1, 2]
    assert ops.rotary_axes((4, 2, 2), "cpu", interleaved=True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    for bad in ((), (1, -1)):
        with pytest.raises(ValueError):
            ops.rotary_axes(bad, "cpu")


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 4, 128)
    pos = torch.zeros(1, 4, dtype=torch.int32)
    rope = ops.Rotary(ops.rotary_frequencies(128, device="cpu"))
    with pytest.raises(ValueError):
        ops.rotary(x, pos, rope)
    with pytest.raises(ValueError):
        ops.kv_append_rotary_paged(x, x, x, x, pos)
    with pytest.raises(ValueError):
        ops.dequantize_q8(torch.zeros(1, 16, 128, dtype=torch.int8), torch.zeros(1, 1))
