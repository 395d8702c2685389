"""What goes wrong inside attention over 8-bit pages is told without a status tensor: last_status() reads the device's
own word, and PagedKVCache needs no more than that."""
import os
import subprocess
import sys

import pytest
import torch

from leankv_b200 import attention
from leankv_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _problem(n, D=128, H=1, P=16, pages=8):
    g = torch.Generator(device=DEV).manual_seed(n + D)
    kp, vp = (torch.randint(-127, 128, (pages, H, P, D), dtype=torch.int8, device=DEV, generator=g) for _ in range(2))
    ks, vs = (torch.rand(pages, H, P // 16, device=DEV, generator=g) / 100 for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, pages)
    q = torch.randn(1, 4 * H, n, D, device=DEV, generator=g).bfloat16()
    return q, kp, vp, ks, vs, table, torch.tensor([pages * P], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [1, 20, 130])   # rows for each of the three kernels
def test_bad_page_without_a_status_tensor(n, D):
    q, kp, vp, ks, vs, table, lens = _problem(n, D)
    attention.last_status()   # whatever calls before have raised
    attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens)
    assert attention.last_status() == 0
    bad = table.clone()
    bad[0, 3] = 8
    attention.attention_q8_paged(q, kp, vp, ks, vs, bad, lens)
    attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens)   # a good call does not hide it
    assert attention.last_status(0) == 1
    assert attention.last_status("cuda") == 0   # asking clears it
    own = torch.zeros(1, dtype=torch.int32, device=DEV)
    attention.attention_q8_paged(q, kp, vp, ks, vs, bad, lens, status=own)
    assert int(own.item()) == 1 and attention.last_status() == 0   # a call's own word is the only one raised


def test_bound_of_the_lengths_without_a_status_tensor():
    q, kp, vp, ks, vs, table, lens = _problem(130)
    attention.last_status()
    attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, max_kv_len=100)
    assert attention.last_status() == 1


def test_cache_tells():
    cache = PagedKVCache(1, 2, 128, num_pages=8, page_size=16, max_seqs=1, k_bits=8)
    s = cache.add_sequence()
    step = cache.batch([s], 40)
    k = torch.randn(1, 2, 40, 128, device=DEV).bfloat16()
    cache.append(step, 0, k, k)
    q = torch.randn(1, 8, 40, 128, device=DEV).bfloat16()
    attention.last_status()
    good = cache.attention(step, 0, q)
    assert attention.last_status() == 0
    step.table[0, 1] = 8
    assert not torch.equal(cache.attention(step, 0, q), good)
    assert attention.last_status() == 1


def test_replayed_graph_tells():
    q, kp, vp, ks, vs, table, lens = _problem(1)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, out=out)
    attention.last_status()
    graph.replay()
    assert attention.last_status() == 0
    table[0, 2] = -5
    graph.replay()
    assert attention.last_status() == 1
    table[0, 2] = 2
    graph.replay()
    assert attention.last_status() == 0


FIRST = """
import torch
from leankv_b200 import attention
g = torch.Generator(device="cuda").manual_seed(1)
kp, vp = (torch.randint(-127, 128, (8, 1, 16, 128), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
ks = torch.full((8, 1, 1), 0.01, device="cuda")
table = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
lens = torch.tensor([128], dtype=torch.int32, device="cuda")
q = torch.randn(1, 4, 1, 128, device="cuda", generator=g).bfloat16()
out = torch.empty_like(q)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    attention.attention_q8_paged(q, kp, vp, ks, ks, table, lens, out=out)
graph.replay()
assert attention.last_status() == 0
assert torch.equal(out, attention.attention_q8_paged(q, kp, vp, ks, ks, table, lens))
table[0, 1] = 99
graph.replay()
assert attention.last_status() == 1 and attention.last_status() == 0
print("told")
"""


def test_first_call_of_a_process_is_a_captured_one():
    run = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "told", run.stdout + run.stderr
