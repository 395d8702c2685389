"""Calls after cudaDeviceReset, which ends the process's own context: the library keeps nothing of the old one.  In a process of its own,
through the C entry points, as torch does not outlive a reset."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
import ctypes as C, glob, os, sys
import numpy as np
import torch
from leankv_b200 import _lib as L, attention, ops

lib = L.load()
found = glob.glob(os.path.join(os.path.dirname(torch.__file__), "..", "nvidia", "cuda_runtime", "lib", "libcudart.so.12"))
rt = C.CDLL((found + ["/usr/local/cuda/lib64/libcudart.so.12"])[0])
H, D, P, PAGES, CAP = 2, 128, 16, 8, 128


def ok(code):
    assert code == 0, (code, lib.tq_last_error_string())


class Device:
    "Arrays in device memory, by name."
    def __init__(self, **arrays):
        self.of = {}
        for name, a in arrays.items():
            p = C.c_void_p()
            ok(rt.cudaMalloc(C.byref(p), C.c_size_t(a.nbytes)))
            ok(rt.cudaMemcpy(p, a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes), 1))
            self.of[name] = (p, a)

    def __getitem__(self, name):
        return self.of[name][0].value

    def get(self, name):
        p, a = self.of[name]
        out = np.empty_like(a)
        ok(rt.cudaMemcpy(out.ctypes.data_as(C.c_void_p), p, C.c_size_t(a.nbytes), 2))
        return out


def status():
    word = C.c_int32(-1)
    ok(lib.tq_attention_q8_last_status(C.byref(word), None))
    return word.value


def select(rng):
    d = Device(w=rng.random((PAGES, H, P), dtype=np.float32), table=np.array([[0, 5, 2, 99, 1, 3, 4, 6]], np.int32),
               lens=np.array([CAP], np.int32), out=np.zeros((1, H, 20), np.int32))
    pages = ops._PAGES.pack(d["table"], PAGES, PAGES, P)
    ok(lib.tq_select_tokens_cuda(ops._SELECT.pack(1, H, d["w"], d["lens"], 0, 20, 2, 3, 0, d["out"], 0), pages, None))
    ok(rt.cudaDeviceSynchronize())
    assert status() == 1 and status() == 0          # page 99 is outside the pool
    return [d.get("out")]


def attend(rng):
    out = []
    for n in (1, 3, 20, 60, 300):                    # few rows, converting and tile kernels; trees and weights beside them
        words = -(-n // 32)
        code = lambda: rng.integers(-127, 128, (PAGES * 4, H, P, D)).astype(np.int8)   # noqa: E731
        scale = lambda: rng.random((PAGES * 4, H, P // 16), dtype=np.float32) / 60     # noqa: E731
        mask = rng.integers(0, 1 << 31, (1, n, words)).astype(np.int32)
        ws = 1 << 26
        d = Device(q=rng.standard_normal((1, 4 * H, n, D), dtype=np.float32), k=code(), v=code(), ks=scale(), vs=scale(), mask=mask,
                   table=np.arange(4 * PAGES, dtype=np.int32)[None], lens=np.array([500], np.int32), o=np.zeros((1, 4 * H, n, D), np.float32),
                   t=np.zeros((1, 4 * H, n, D), np.float32), lse=np.zeros((1, 4 * H, n), np.float32), w=np.zeros((PAGES * 4, H, P), np.float32),
                   ws=np.zeros(ws, np.uint8))
        pages = ops._PAGES.pack(d["table"], 4 * PAGES, 4 * PAGES, P)
        args = lambda o: attention._ATTN_Q8.pack(1, 4 * H, H, D, n, d["q"], 0, 4 * H * n * D, n * D, D, d[o], 0, 4 * H * n * D, n * D, D, d["k"],   # noqa: E731
                                                 d["ks"], d["v"], d["vs"], d["lens"], 0, 0, 0.0, 1, 1, 1, d["lse"], 0, d["ws"], ws)
        ok(lib.tq_attention_q8_tree_paged_cuda(args("t"), pages, attention._MASK.pack(d["mask"], 0), None))
        ok(lib.tq_attention_q8_paged_cuda(args("o"), pages, None))
        ok(lib.tq_attention_weights_paged_cuda(attention._WEIGHTS.pack(1, 4 * H, H, D, n, d["q"], 0, 4 * H * n * D, n * D, D, d["k"], 8, d["ks"],
                                                                       d["lens"], 0, d["lse"], 0, 0, 0.0, 1, 1, 1.0, 0, d["w"], 0, d["ws"], ws),
                                               pages, None))
        ok(rt.cudaDeviceSynchronize())
        assert status() == 0
        out += [d.get(x) for x in ("o", "t", "lse", "w")]
    return out


runs = {"select": select, "attend": attend}
results = []
for _ in range(3):
    results.append(runs[sys.argv[1]](np.random.default_rng(1)))
    ok(rt.cudaDeviceReset())
for other in results[1:]:
    assert all(np.array_equal(a, b) for a, b in zip(results[0], other))
assert all(np.isfinite(a).all() and a.any() for a in results[0])
print("done")
"""


def _run(what):
    r = subprocess.run([sys.executable, "-c", PROGRAM, what], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True,
                       timeout=240)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout[-1500:] + r.stderr[-3000:]


def test_the_word_of_calls_without_a_status():
    _run("select")


def test_kernels_with_more_shared_memory_than_the_default():
    _run("attend")
