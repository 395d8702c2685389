"""Pools and rows whose offsets pass 32 bits: the same pages at the start and at the end of a pool of more than 2^32 bytes,
and rows more than 2^32 bytes into a tensor, give the same results bit for bit."""
import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
P, H = 64, 8


def _far_pool(D, seed):
    """int8 pool of a little more than 2^32 codes and its scales; only the first and last 16 pages hold anything."""
    pages = (1 << 32) // (H * P * D) + 16
    g = torch.Generator(device=DEV).manual_seed(seed)
    pool = torch.zeros(pages, H, P, D, dtype=torch.int8, device=DEV)
    scale = torch.zeros(pages, H, P // 16, device=DEV)
    pool[:16] = torch.randint(-127, 128, (16, H, P, D), dtype=torch.int8, device=DEV, generator=g)
    scale[:16] = torch.rand(16, H, P // 16, device=DEV, generator=g) / 100
    pool[-16:], scale[-16:] = pool[:16], scale[:16]
    return pool, scale


@pytest.mark.parametrize("D", [128, 256])
def test_attention_and_append(D):
    kp, ks = _far_pool(D, 1)
    vp, vs = _far_pool(D, 2)
    near = torch.arange(16, dtype=torch.int32, device=DEV).flip(0).view(2, 8).contiguous()
    far = near + (kp.shape[0] - 16)
    lens = torch.tensor([500, 333], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    for n in (1, 5, 20, 130):   # each kernel
        q = torch.randn(2, 4 * H, n, D, device=DEV, generator=g).bfloat16()
        a, b = (attention.attention_q8_paged(q, kp, vp, ks, vs, t, lens) for t in (near, far))
        assert torch.equal(a, b) and a.any()
    k, v = (torch.randn(2, H, 30, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    pos = torch.tensor([480, 37], dtype=torch.int32, device=DEV)
    before = kp[16:-16].any(), kp[-16:].clone()
    for t in (near, far):
        ops.kv_append_rotary_paged(k, v, kp, vp, t, pos, rope=rope, k_scale=ks, v_scale=vs)
    assert torch.equal(kp[:16], kp[-16:]) and torch.equal(vp[:16], vp[-16:])
    assert torch.equal(ks[:16], ks[-16:]) and torch.equal(vs[:16], vs[-16:])
    assert not torch.equal(kp[-16:], before[1]) and not before[0] and not kp[16:-16].any()
    tail = ops.dequantize_q8(kp, ks, torch.float16)[-16:]
    assert torch.equal(tail, ops.dequantize_q8(kp[-16:], ks[-16:], torch.float16))


@pytest.mark.parametrize("bits", [2, 4])
def test_append_into_tq_pools(bits):
    D = 256
    kb = ops.BLOCK_BYTES[bits]
    pages = (1 << 32) // (H * P * D // 32 * kb) + 16
    kp = torch.zeros(pages, H, P, D // 32, kb, dtype=torch.uint8, device=DEV)
    vp = torch.zeros(pages, H, P, D // 32, 18, dtype=torch.uint8, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(4)
    k, v = (torch.randn(1, H, 90, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    near = torch.tensor([[3, 0]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([11], dtype=torch.int32, device=DEV)
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    for t in (near, near + (pages - 16)):
        ops.kv_append_rotary_paged(k, v, kp, vp, t, pos, rope=rope)
    assert torch.equal(kp[:16], kp[-16:]) and torch.equal(vp[:16], vp[-16:]) and kp[:16].any() and vp[:16].any()
    assert not kp[16:-16].any() and not vp[16:-16].any()


def test_rows_far_into_a_tensor():
    """Tokens, heads and sequences more than 2^32 bytes apart, as sources and as destinations."""
    D, step = 128, (1 << 31) + 1024   # elements of 2 bytes
    memory = torch.empty(2 * step + 4096, dtype=torch.bfloat16, device=DEV)
    other = torch.empty_like(memory)
    rope = ops.Rotary(ops.rotary_frequencies(D, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(5)
    kp, vp = (torch.randint(-127, 128, (4, 1, P, D), dtype=torch.int8, device=DEV, generator=g) for _ in range(2))
    ks, vs = (torch.rand(4, 1, P // 16, device=DEV, generator=g) / 100 for _ in range(2))
    for shape in ((3, 2, 2, D), (2, 3, 2, D), (2, 2, 3, D)):
        where = shape.index(3)
        strides = [D, 2 * D, 4 * D]
        strides = strides[:where] + [step] + strides[where:2] + [1]
        x = torch.randn(shape, device=DEV, generator=g).bfloat16()
        far, out = memory.as_strided(shape, strides), other.as_strided(shape, strides)
        far.copy_(x)
        pos = torch.randint(0, 1000, (shape[0], shape[2]), dtype=torch.int32, device=DEV, generator=g)
        want = ops.rotary(x, pos, rope)
        assert torch.equal(ops.rotary(far, pos, rope), want)
        assert torch.equal(ops.rotary(far, pos, rope, out=out), want)
        table = torch.tensor([[2, 0, 3, 1]] * shape[0], dtype=torch.int32, device=DEV)
        lens = torch.tensor([200, 150, 9][:shape[0]], dtype=torch.int32, device=DEV)
        want = attention.attention_q8_paged(x, kp, vp, ks, vs, table, lens)
        assert torch.equal(attention.attention_q8_paged(far, kp, vp, ks, vs, table, lens), want)
        assert torch.equal(attention.attention_q8_paged(far, kp, vp, ks, vs, table, lens, out=out), want)
