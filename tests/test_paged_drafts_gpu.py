"""Drafted tokens that are rejected: the step is not committed, a batch of the accepted count is, and later rows take the
rejected ones' slots.  TQ pages end as if the rejected rows had never been; 8-bit blocks may keep a grown scale, so their
attention is held to the 8-bit tier's usual error."""
import math

import pytest
import torch

from leankv_b200 import ops
from leankv_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("k_bits", [2, 3, 4, 8])
def test_rejected_drafts(k_bits):
    D, hk, grp = 128, 2, 4
    make = lambda: PagedKVCache(1, hk, D, num_pages=20, page_size=16, max_seqs=2, k_bits=k_bits)   # noqa: E731
    one, two = make(), make()
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    seqs = [one.add_sequence(), one.add_sequence()]
    assert seqs == [two.add_sequence(), two.add_sequence()]
    g = torch.Generator(device=DEV).manual_seed(k_bits)
    rand = lambda n, h: torch.randn(2, h, n, D, device=DEV, generator=g).bfloat16()   # noqa: E731
    held = [[], []]
    for n, accepted in ((13, [13, 13]), (5, [2, 4]), (5, [0, 5]), (5, [1, 1]), (1, [1, 1])):
        k, v = rand(n, hk), rand(n, hk)
        drafts = one.batch(seqs, n)
        one.append(drafts, 0, k, v, rope=rope)
        keep = one.batch(seqs, accepted)          # in place of the drafts' commit; their rows are in the pages already
        assert keep.pos.tolist() == drafts.pos.tolist()
        one.commit(keep)
        step = two.batch(seqs, accepted)          # as if the others had never been
        m = max(accepted)
        two.append(step, 0, k[:, :, :m], v[:, :, :m], rope=rope)
        two.commit(step)
        where = (step.pos[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)).contiguous()
        kr = ops.rotary(k.float(), where, rope)
        for b, c in enumerate(accepted):
            held[b].append((kr[b, :, :c], v[b, :, :c].float()))
    assert [one.seq_len(s) for s in seqs] == [two.seq_len(s) for s in seqs] == [17, 24]
    q = rand(1, hk * grp)[:, :, 0].contiguous()
    # the last token again, alone, in both (one page each so far, or two)
    outs = []
    for c in (one, two):
        step = c.batch(seqs, 0)
        outs.append(c.attention(step, 0, q))
    if k_bits != 8:
        assert torch.equal(outs[0], outs[1])
        return
    for b in range(2):
        K, V = (torch.cat(t, 1).double().repeat_interleave(grp, 0) for t in zip(*held[b]))
        p = torch.softmax((q[b].double()[:, None] @ K.transpose(1, 2)) / math.sqrt(D), -1)
        want = (p @ V)[:, 0]
        # codes are off by half a step of a block's largest of 16 D values, about 4.5 deviations / 127, once when written and
        # once more for each time that the scale grew (as in the other tests of this tier: 0.01 deviations each)
        assert float((outs[0][b].double() - want).norm() / want.norm()) < 0.03
