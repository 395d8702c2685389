"""PagedKVCache.attention of one row per sequence in steps of unequal counts: the row of a sequence without a new token is
padding and gives zeros in every tier; the others' rows are those of a step without the padding."""
import pytest
import torch

from leankv_b200 import attention, ops
from leankv_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("k_bits", [2, 3, 4, 8])
@pytest.mark.parametrize("counts", [[1, 0, 1], [0, 3, 0], [5, 0, 2]])
def test_sequences_without_a_new_token(k_bits, counts, D):
    hk, grp, B = 2, 4, 3
    cache = PagedKVCache(1, hk, D, num_pages=30, page_size=16, max_seqs=B, k_bits=k_bits)
    seqs = [cache.add_sequence() for _ in range(B)]
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(D + k_bits)
    rand = lambda h, n: torch.randn(B, h, n, D, device=DEV, generator=g).bfloat16()   # noqa: E731
    first = cache.batch(seqs, [40, 17, 33])
    cache.append(first, 0, rand(hk, 40), rand(hk, 40), rope=rope)
    cache.commit(first)
    held = [cache.seq_len(s) for s in seqs]
    step = cache.batch(seqs, counts)
    cache.append(step, 0, rand(hk, step.n_new), rand(hk, step.n_new), rope=rope)
    assert step.kv_len.tolist() == [h + c for h, c in zip(held, counts)]
    q = rand(hk * grp, 1)[:, :, 0].contiguous()
    out = torch.full_like(q, 7.0)
    assert cache.attention(step, 0, q, out=out).data_ptr() == out.data_ptr()
    if k_bits == 8:
        want = attention.attention_q8_paged(q, cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0], step.table,
                                            step.kv_len, max_kv_len=step.max_kv_len)
    else:
        want = attention.decode_attention_paged(q, cache.k[0], cache.v[0], step.table, step.kv_len, max_kv_len=step.max_kv_len,
                                                out_dtype=q.dtype)
    for b, c in enumerate(counts):
        assert torch.equal(out[b], want[b] if c else torch.zeros_like(out[b]))
    assert attention.last_status() == 0
    cache.commit(step)
    assert [cache.seq_len(s) for s in seqs] == [h + c for h, c in zip(held, counts)]
