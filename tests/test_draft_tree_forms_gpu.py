"""The forms of the tree attention and of the sums of weights that sizes beyond the other tests' choose: two row tiles a CTA, heads of 256
in one tile of rows, several passes of the work memory.  Tolerances are those of the tests whose comparison is used."""
import pytest
import torch

import test_attention_weights_gpu as weights
import test_draft_tree_gpu as tree
from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _trees(B, n, seed):
    parents = tree._parents(B, n, seed)
    return tree._ancestors(parents), ops.draft_tree(parents.to(DEV))


@pytest.mark.parametrize("n,grp", [(64, 8), (57, 8), (120, 4), (450, 1)])
def test_two_row_tiles(n, grp):
    # from 449 rows on with as many (sequence, KV head)s that two tiles of rows a CTA leave no SM idle
    B = 19
    lens = [n + 37 * (i % 7) + (500 if i == 3 else 0) for i in range(B)]
    q_len = [n - (i % 3) * (n // 3) for i in range(B)]
    lens[1], lens[2], q_len[2] = n, n - 5, n
    seen, mask = _trees(B, n, n)
    tree._check(B, 2, grp, n, 128, 16, torch.bfloat16, lens, q_len, seen, mask, seed=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,grp", [(1, 8), (4, 2), (8, 1), (2, 3)])
def test_heads_of_256_in_one_tile_of_rows(n, grp, dtype):
    lens, q_len = [700 + n, 17, n, max(1, n - 1), 200], [n, n, n, n, 1]
    seen, mask = _trees(5, n, n)
    tree._check(5, 2, grp, n, 256, 32, dtype, lens, q_len, seen, mask, seed=grp)


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (256, torch.float16)])
def test_several_passes_of_the_work_memory(D, dtype, monkeypatch):
    """Tables for sequences so long that the work memory holds the tiles of some (sequence, KV head)s at a time."""
    columns = 1 << 14     # 262144 tokens of 513 or 1025 bytes of tiles: 7 or 3 of 10 at a time
    call = attention.attention_q8_paged
    need = []

    def wide(q, kp, vp, ks, vs, table, kv_len, **kw):
        more = torch.zeros(len(table), columns, dtype=torch.int32, device=DEV)
        more[:, : table.shape[1]] = table
        key = len(ops._work_sizes)
        out = call(q, kp, vp, ks, vs, more, kv_len, **kw)
        need.extend(list(ops._work_sizes.values())[key:])
        return out
    monkeypatch.setattr(attention, "attention_q8_paged", wide)
    monkeypatch.setattr(ops, "_work_sizes", {})
    n, grp = 60, 8
    seen, mask = _trees(5, n, n)
    tree._check(5, 2, grp, n, D, 16, dtype, [600 + n, 37, n, n + 1, 300], [n, 20, n, n, n // 2], seen, mask, seed=D)
    assert need and need[0] < 10 * columns * 16 * 4 * D


@pytest.mark.parametrize("n,grp", [(3, 3), (5, 4), (2, 16), (32, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_of_up_to_32_rows_of_256(n, grp, causal):
    weights._check(8, 4, 2, grp, n, 256, 32, torch.bfloat16, [900, n, 20 + n, 301], q_len=[n, n, n - 1, n], fresh=[900 - n, 0, 7, 100], decay=0.5,
                   causal=causal, seed=n)


def test_weights_in_several_passes_of_the_work_memory():
    B, grp, n = 90, 8, 4096          # 46080 tiles of 64 rows of 25 KB in 1 GiB
    weights._check(8, B, 1, grp, n, 128, 16, torch.bfloat16, [20 + i % 13 for i in range(B)], causal=False, seed=3)


@pytest.mark.parametrize("B,n,grp,D,dtype", [(1, 10, 4, 128, torch.bfloat16), (16, 26, 4, 128, torch.bfloat16), (3, 63, 8, 256, torch.float16),
                                             (19, 64, 8, 128, torch.bfloat16), (2, 1, 8, 256, torch.float32)])
def test_the_same_call_gives_the_same_bits(B, n, grp, D, dtype):
    H, P, L = 2, 16, 1200
    per = L // P
    kp, ks = tree._pools(B * per, H, P, D, 1)
    vp, vs = tree._pools(B * per, H, P, D, 2)
    table = torch.randperm(B * per, generator=torch.Generator().manual_seed(B)).view(B, per).to(torch.int32).to(DEV)
    lens = torch.tensor([max(n, L - 61 * i) for i in range(B)], dtype=torch.int32, device=DEV)
    q = torch.randn(B, n, H * grp, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).to(dtype).transpose(1, 2)
    mask = ops.draft_tree(tree._parents(B, n, n).to(DEV))
    first = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, tree=mask, return_lse=True)
    for _ in range(5):
        again = attention.attention_q8_paged(q, kp, vp, ks, vs, table, lens, tree=mask, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
