"""Many steps of drafted trees over 8-bit pages: what the pages hold after each append and each accepted path equals the two documented
rules one after another, and stays within the sum of their roundings of the rows that were given.

The block that a sequence's last tokens lie in is written by every step: the append may grow its scale for nodes that are then rejected,
and the accepted path's move sets it back to what its rows need.  Both round the block's earlier rows, each time by at most half of the
new scale; a block that is full is not touched again.  The bound of each row is that sum, with 2^-12 of it for the roundings of float32
(127 times 2^-23 for each product)."""
import pytest
import torch

import test_kv_move_gpu as moves
from leankv_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, H, D, P, PER, NODES, STEPS = 3, 2, 128, 16, 12, 26, 45
T = P * PER


def _rows(pool):
    return pool.view(B, PER, H, P, -1).transpose(1, 2).flatten(2, 3).squeeze(-1)     # [B, H, slots, ...]


def _store(pool, rows):
    pool.copy_(rows.reshape(B, H, PER, P, *pool.shape[3:]).transpose(1, 2).reshape(pool.shape))


class Side:
    """The pages of K or of V, the values that were given and what the rules allow them to be off by."""

    def __init__(self):
        self.pool, self.scale = torch.zeros(B * PER, H, P, D, dtype=torch.int8, device=DEV), torch.zeros(B * PER, H, 1, device=DEV)
        self.true, self.off = torch.zeros(B, H, T, D, device=DEV), torch.zeros(B, H, T, device=DEV).double()

    def append(self, rows, pos):
        """The append's rule: codes and scales that the pages have to hold then."""
        code, scale = _rows(self.pool).clone().float(), self.scale.view(B, PER, H).transpose(1, 2).clone()
        for b, first in enumerate(pos):
            for block in range(first // 16, (first + NODES - 1) // 16 + 1):
                lo, hi = max(first, 16 * block), min(first + NODES, 16 * block + 16)
                old = scale[b, :, block].clone() if lo > 16 * block else torch.zeros(H, device=DEV)
                x = rows[b, :, lo - first: hi - first]
                new = torch.maximum(old, x.abs().amax((-1, -2)) * torch.tensor(1.0 / 127.0, device=DEV))
                inv = 1.0 / new
                older = slice(16 * block, lo)
                code[b, :, older] = torch.round(code[b, :, older] * (old * inv)[:, None, None])
                self.off[b, :, older] += 0.5 * torch.where(new == old, 0.0, new).double()[:, None]
                code[b, :, lo:hi] = torch.round(x * inv[:, None, None]).clamp(-127, 127)
                self.true[b, :, lo:hi], self.off[b, :, lo:hi] = x, 0.5 * new.double()[:, None]
                scale[b, :, block] = new
        return code, scale

    def moved(self, table, src, first, count):
        code, scale, _, left = moves._expected(self.pool, self.scale, None, table, table, src, first, count, True)
        assert left == 0
        now = scale.view(B, PER, H).transpose(1, 2).double()
        for b in range(B):
            at = src[b, : count[b]].long()
            to = torch.arange(first[b], first[b] + count[b], device=DEV)
            self.true[b, :, to], self.off[b, :, to] = self.true[b, :, at], self.off[b, :, at]
            if count[b] and not torch.equal(at, to):
                last = first[b] + count[b]
                for block in range(first[b] // 16, (last - 1) // 16 + 1):
                    held = slice(16 * block, min(last, 16 * block + 16))     # rounded again, unless all its rows stay or have one scale
                    self.off[b, :, held] += 0.5 * now[b, :, block, None]
        return code, scale

    def check(self, ends):
        value = _rows(self.pool).double() * self.scale.view(B, PER, H).transpose(1, 2).double().repeat_interleave(16, -1)[..., None]
        off = (value - self.true.double()).abs().amax(-1)
        for b, end in enumerate(ends):
            assert bool((off[b, :, :end] <= self.off[b, :, :end] * (1 + 2.0 ** -12)).all())
        return value


def _size(gen, *shape):
    return torch.exp(0.6 * torch.randn(*shape, 1, device=DEV, generator=gen))     # rows of unlike size


def test_many_steps():
    gen = torch.Generator(device=DEV).manual_seed(1)
    cpu = torch.Generator().manual_seed(1)
    table = torch.arange(B * PER, dtype=torch.int32, device=DEV).view(B, PER)
    sides = [Side(), Side()]
    lens = [0, 5, 15]
    for step in range(STEPS):
        rows = [torch.randn(B, H, NODES, D, device=DEV, generator=gen) * _size(gen, B, H, NODES) for _ in sides]
        want = [x.append(r, lens) for x, r in zip(sides, rows)]
        pos = torch.tensor(lens, dtype=torch.int32, device=DEV)
        (k, v) = sides
        ops.kv_append_rotary_paged(rows[0], rows[1], k.pool, v.pool, table, pos, k_scale=k.scale, v_scale=v.scale, rotate=False)
        for x, (code, scale) in zip(sides, want):
            for b, first in enumerate(lens):
                assert torch.equal(_rows(x.pool)[b, :, :first + NODES].float(), code[b, :, :first + NODES])
                blocks = -(-(first + NODES) // 16)
                assert torch.equal(x.scale.view(B, PER, H).transpose(1, 2)[b, :, :blocks], scale[b, :, :blocks])
        count = [int(torch.randint(0, 7, (1,), generator=cpu)) if lens[b] < T - NODES - 7 else 0 for b in range(B)]
        path = torch.stack([torch.randperm(NODES, generator=cpu)[:6].sort().values for _ in range(B)])
        src = (path + torch.tensor(lens)[:, None]).to(torch.int32).to(DEV)
        want = [x.moved(table, src, lens, count) for x in sides]
        ops.kv_move_paged(k.pool, v.pool, table, src, first=pos, count=torch.tensor(count, dtype=torch.int32, device=DEV), k_scale=k.scale,
                          v_scale=v.scale)
        lens = [n + c for n, c in zip(lens, count)]
        for x, (code, scale) in zip(sides, want):
            assert torch.equal(x.pool, code) and torch.equal(x.scale, scale)
            x.check(lens)
    assert min(lens) > 100
