"""Prompts over 8-bit pages whose work memory holds the tiles of some (sequence, KV head) pairs only, so that a call
runs in several passes, the last one of fewer pairs: wide page tables over short sequences, against the formula with
the tolerances of test_attention_q8_gpu."""
import pytest
import torch
from test_attention_q8_gpu import _check, _pools, _q, _table

from leankv_b200 import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
GIB = 1 << 30


def _wide(table, P, tokens):
    """The same pages in a table that has room for `tokens` tokens of each sequence."""
    wide = torch.full((table.shape[0], tokens // P), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    return wide


# tokens: the bound that leaves room for 3 pairs (1 in the last case); rows for one and for two row tiles a CTA
@pytest.mark.parametrize("D,dtype,grp,n,top,tokens,at_a_time", [
    (128, torch.bfloat16, 4, 120, 700, 1 << 19, 3), (128, torch.float16, 4, 120, 300, 1 << 19, 3),
    (256, torch.float16, 4, 120, 700, 1 << 18, 3), (256, torch.bfloat16, 8, 60, 200, 1 << 18, 3),
    (128, torch.bfloat16, 4, 1700, 2000, 1 << 19, 3), (128, torch.bfloat16, 3, 150, 500, 1 << 20, 1)])
def test_several_passes_match_formula(D, dtype, grp, n, top, tokens, at_a_time):
    B, H, P = 5, 1, 64
    assert GIB // (tokens * (4 * D + 1)) == at_a_time   # two f16 tiles, 16 bytes for 16 tokens
    per = -(-top // P)
    kp, ks = _pools(B * per + 3, H, P, D, 1)
    vp, vs = _pools(B * per + 3, H, P, D, 2)
    table = _wide(_table(B, per, B * per + 3, 3), P, tokens)
    lens = torch.tensor([top, 129, 0, n // 2 + 1, top - 5], dtype=torch.int32, device=DEV)
    q = _q(B, H * grp, n, D, dtype, n)
    _check(q, kp, vp, ks, vs, table, lens)
    ql = torch.tensor([n, n // 3, 3, n // 2 + 1, 0], dtype=torch.int32, device=DEV)
    _check(q, kp, vp, ks, vs, table, lens, q_len=ql)


def test_several_heads_and_a_replayed_graph():
    """Passes that end inside a sequence's heads; the graph's passes share their own work memory."""
    B, H, grp, n, D, P, tokens = 3, 5, 4, 120, 128, 64, 1 << 18
    assert GIB // (tokens * (4 * D + 1)) == 7
    kp, ks = _pools(40, H, P, D, 4)
    vp, vs = _pools(40, H, P, D, 5)
    table = _wide(_table(B, 12, 40, 6), P, tokens)
    lens = torch.tensor([768, 333, 120], dtype=torch.int32, device=DEV)
    q = _q(B, H * grp, n, D, torch.bfloat16, 7)
    want = _check(q, kp, vp, ks, vs, table, lens)[0]
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, out=out)
    for L in (768, 200, 0):
        lens[0] = L
        out.zero_()
        graph.replay()
        assert torch.equal(out, attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens))
