"""Rotary and 8-bit page entry points without a GPU: statuses of refused arguments (set before any device
work), the helpers that build frequencies and axes, and the argument blocks' layouts."""
import subprocess

import pytest
import torch

from leankv_b200 import _lib as L
from leankv_b200 import ops


ROPE = ["inv_freq", "axis", "positions", "n_axes", "rotary_dim", "interleaved", "inverse", "scale"]
HEADS = ["src", "dst", "heads", "s0", "s1", "s2", "d0", "d1", "d2"]


def _rope(**kw):
    base = dict(inv_freq=64, axis=0, positions=64, n_axes=1, rotary_dim=64, interleaved=0, inverse=0, scale=1.0)
    return tuple({**base, **kw}[n] for n in ROPE)


def _heads(**kw):
    base = dict(src=64, dst=64, heads=2, s0=1024, s1=128, s2=256, d0=1024, d1=128, d2=256)
    return tuple({**base, **kw}[n] for n in HEADS)


@pytest.mark.parametrize("rope,dtype,batch,n,D,x,status", [
    (dict(rotary_dim=24), 1, 1, 1, 64, {}, 1), (dict(rotary_dim=128), 1, 1, 1, 64, {}, 1),
    (dict(inv_freq=0), 1, 1, 1, 64, {}, 1), (dict(positions=0), 1, 1, 1, 64, {}, 1),
    (dict(n_axes=0), 1, 1, 1, 64, {}, 1), (dict(scale=float("inf")), 1, 1, 1, 64, {}, 1),
    (dict(inv_freq=68), 1, 1, 1, 64, {}, 3), (dict(positions=66), 1, 1, 1, 64, {}, 3),
    ({}, 5, 1, 1, 64, {}, 1), ({}, 1, -1, 1, 64, {}, 1), ({}, 1, 1, -1, 64, {}, 1), ({}, 1, 1, 1 << 31, 64, {}, 1),
    ({}, 1, 1, 1, 68, {}, 2), ({}, 1, 1, 1, 520, {}, 2), ({}, 1, 1, 1, 64, dict(heads=0), 1),
    ({}, 1, 1, 1, 64, dict(src=0), 1), ({}, 1, 1, 1, 64, dict(src=72), 3),
    ({}, 1, 1, 1, 64, dict(s2=132, dst=128), 3),
    ({}, 1, 1, 1, 64, dict(s2=512), 1),
    ({}, 1, 0, 1, 64, {}, 0), ({}, 1, 1, 0, 64, {}, 0)])
def test_rotary_statuses(rope, dtype, batch, n, D, x, status):
    lib = L.load()
    got = lib.tq_rotary_cuda(ops._ROPE.pack(*_rope(**rope)), dtype, batch, n, D, ops._HEADS.pack(*_heads(**x)), None, None)
    assert got == status
    assert status == 0 or lib.tq_last_error_string()


APPEND = ["batch", "n_kv_heads", "head_dim", "n_new", "dtype", "k", "v", "q", "rope", "k_pool", "k_type", "k_scale",
          "v_pool", "v_type", "v_scale", "pos", "new_len", "rotate", "overflow"]


def _append(**kw):
    h = _heads(dst=0)
    base = dict(batch=1, n_kv_heads=2, head_dim=128, n_new=1, dtype=1, k=h, v=h, q=ops._NO_HEADS,
                rope=_rope(rotary_dim=128, positions=0), k_pool=64, k_type=8, k_scale=64, v_pool=64, v_type=8, v_scale=64,
                pos=0, new_len=0, rotate=1, overflow=0)
    flat = []
    for name in APPEND:
        value = {**base, **kw}[name]
        flat += value if isinstance(value, tuple) else [value]
    return ops._APPEND.pack(*flat)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), 1), (dict(n_kv_heads=0), 1), (dict(head_dim=64), 2), (dict(k_type=3), 2), (dict(k_type=5), 2),
    (dict(v_type=4), 2), (dict(rope=_rope(rotary_dim=128, inverse=1)), 1),
    (dict(rope=_rope(rotary_dim=128, positions=0, n_axes=3)), 1),
    (dict(rope=ops._NO_ROPE, q=_heads()), 1), (dict(k=_heads(heads=3)), 1), (dict(v=_heads(src=0)), 1),
    (dict(q=_heads(dst=0)), 1), (dict(k_scale=0), 1), (dict(v_pool=0), 1), (dict(k_pool=72), 3),
    (dict(v_scale=66), 3), (dict(pos=66), 3), (dict(q=_heads(heads=-1)), 1), (dict(n_new=0), 0), (dict(batch=0), 0)])
def test_append_statuses(change, status):
    fn = L.load().tq_kv_append_rotary_paged_cuda
    assert fn(_append(**change), ops._PAGES.pack(64, 4, 8, 16), None) == status
    assert fn(_append(), ops._PAGES.pack(64, 4, 8, 24), None) == 1
    assert fn(_append(), None, None) == 1


ATTN = ["batch", "n_q_heads", "n_kv_heads", "head_dim", "n_new", "q", "q_dtype", "qs0", "qs1", "qs2", "out", "out_dtype", "os0",
        "os1", "os2", "k", "ks", "v", "vs", "kv_len", "q_len", "max_kv_len", "sm_scale", "causal", "rotate_q", "v_rotated", "lse",
        "status", "workspace", "bytes"]


@pytest.mark.parametrize("change,status", [
    (dict(batch=-1), 1), (dict(n_q_heads=3), 1), (dict(n_kv_heads=0), 1), (dict(head_dim=64), 2), (dict(q_dtype=4), 1),
    (dict(out_dtype=-1), 1), (dict(n_new=-1), 1), (dict(n_new=1 << 30), 2), (dict(max_kv_len=65), 1), (dict(max_kv_len=-1), 1),
    (dict(sm_scale=float("inf")), 1), (dict(q=0), 1), (dict(kv_len=0), 1), (dict(vs=0), 1), (dict(q=72), 3), (dict(qs2=129), 3),
    (dict(os1=4), 3), (dict(k=72), 3), (dict(ks=66), 3), (dict(lse=66), 3), (dict(q_len=65), 3), (dict(n_new=0), 0), (dict(batch=0), 0),
    (dict(workspace=0), 1), (dict(bytes=16), 1), (dict(workspace=72), 3)])
def test_attention_q8_statuses(change, status):
    from leankv_b200.attention import _ATTN_Q8
    # a batch and a length whose work is split, so that work memory is needed
    base = dict(batch=1, n_q_heads=4, n_kv_heads=2, head_dim=128, n_new=1, q=64, q_dtype=1, qs0=512, qs1=128, qs2=512, out=64,
                out_dtype=1, os0=512, os1=128, os2=512, k=64, ks=64, v=64, vs=64, kv_len=64, q_len=0, max_kv_len=0, sm_scale=0.0,
                causal=1, rotate_q=1, v_rotated=1, lse=0, status=0, workspace=64, bytes=1 << 30)
    pages = ops._PAGES.pack(64, 4, 8, 16) if "max_kv_len" in change else ops._PAGES.pack(64, 4096, 8, 16)
    lib = L.load()
    pack = lambda d: _ATTN_Q8.pack(*(d[n] for n in ATTN))   # noqa: E731
    assert lib.tq_attention_q8_workspace_size(pack(base), pages if "max_kv_len" not in change else ops._PAGES.pack(64, 4096, 8, 16)) > 16
    assert lib.tq_attention_q8_paged_cuda(pack({**base, **change}), pages, None) == status
    assert lib.tq_attention_q8_paged_cuda(None, pages, None) == 1 and lib.tq_attention_q8_workspace_size(None, pages) == 0


@pytest.mark.parametrize("args,status", [
    ((64, 64, 64, 7, 1, 128), 1), ((64, 64, 64, 0, 1, 64), 2), ((64, 64, 64, 0, -1, 128), 1), ((None, 64, 64, 0, 1, 128), 1),
    ((72, 64, 64, 0, 1, 128), 3), ((64, 66, 64, 0, 1, 128), 3), ((None, None, None, 0, 0, 128), 0)])
def test_dequantize_q8_statuses(args, status):
    assert L.load().tq_dequantize_q8_cuda(*args, None) == status


def test_argument_blocks_match_the_header(tmp_path):
    """Each packed layout against the C structure: a value of its own in every field, read back by a C program."""
    from leankv_b200.attention import _ATTN_Q8
    blocks = {
        "tq_rope": (ops._ROPE, "inv_freq axis positions n_axes rotary_dim interleaved inverse scale"),
        "tq_head_rows": (ops._HEADS, "src dst heads src_stride[0] src_stride[1] src_stride[2] dst_stride[0] dst_stride[1] dst_stride[2]"),
        "tq_kv_pages": (ops._PAGES, "page_table max_pages_per_seq num_pages page_size"),
        "tq_rotary_append_args": (ops._APPEND, " ".join(
            ["batch n_kv_heads head_dim n_new dtype"]
            + [f"{t}.{f}" for t in "kvq" for f in "src dst heads src_stride[0] src_stride[1] src_stride[2] dst_stride[0] dst_stride[1] dst_stride[2]".split()]
            + [f"rope.{f}" for f in ROPE] + ["k_pool k_type k_scale v_pool v_type v_scale pos new_len rotate overflow"])),
        "tq_attention_q8_args": (_ATTN_Q8, "batch n_q_heads n_kv_heads head_dim n_new q q_dtype q_stride[0] q_stride[1] q_stride[2] "
                                           "out out_dtype out_stride[0] out_stride[1] out_stride[2] k_codes k_scale v_codes v_scale kv_len "
                                           "q_len max_kv_len sm_scale causal rotate_q v_rotated lse status workspace workspace_bytes"),
    }
    for name, (layout, fields) in blocks.items():
        fields = fields.split()
        raw = layout.pack(*range(1, len(fields) + 1))
        src = tmp_path / f"{name}.c"
        src.write_text('#include "leankv_tq.h"\n#include <stdio.h>\n#include <string.h>\nint main(void){\n'
                       f"  static const unsigned char raw[] = {{{', '.join(map(str, raw))}}};\n  {name} a;\n"
                       "  memset(&a, 0, sizeof a); memcpy(&a, raw, sizeof raw);\n  if (sizeof raw > sizeof a) return 1;\n"
                       + "".join(f"  if ((long)a.{f} != {i + 1}) {{ printf(\"{f}\\n\"); return 1; }}\n" for i, f in enumerate(fields))
                       + "  return 0;\n}\n")
        exe = tmp_path / name
        subprocess.run(["gcc", "-I", L.HEADER_DIR, str(src), "-o", str(exe)], check=True)
        run = subprocess.run([str(exe)], capture_output=True, text=True)
        assert run.returncode == 0, (name, run.stdout)


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
