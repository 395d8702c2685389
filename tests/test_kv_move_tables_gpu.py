"""Moving rows to other pages and then, by the same sizes, into a table that is the pages' own: in place, whatever came before."""
import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [8, 3])
def test_the_pages_own_table_is_in_place(bits):
    H, D, P, per, m = 2, 128, 16, 20, 200       # several chunks: they need work memory in place
    g = torch.Generator(device=DEV).manual_seed(bits)
    if bits == 8:
        k, v = (torch.randint(-127, 128, (2 * per, H, P, D), dtype=torch.int8, device=DEV, generator=g) for _ in range(2))
        ks, vs = (torch.rand(2 * per, H, P // 16, device=DEV, generator=g) + 0.5 for _ in range(2))
    else:
        k, v = (torch.randint(0, 256, (2 * per, H, P, D // 32, b), dtype=torch.uint8, device=DEV, generator=g) for b in (14, 18))
        ks = vs = None
    table = torch.arange(per, dtype=torch.int32, device=DEV).view(1, per)
    src = torch.stack([torch.randperm(per * P, device=DEV, generator=g)[:m].sort().values for _ in range(H)])[None].to(torch.int32)

    def moved(to_table):
        pools = [None if t is None else t.clone() for t in (k, v, ks, vs)]
        ops.kv_move_paged(pools[0], pools[1], table, src, k_scale=pools[2], v_scale=pools[3], to_table=to_table)
        return pools
    moved(table + per)
    for a, b in zip(moved(table), moved(None)):
        assert a is None or torch.equal(a, b)
    assert attention.last_status() == 0
