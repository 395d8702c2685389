"""Cases of the rotary, paged-append and 8-bit paged-attention operators: inputs, plain forms, exact values, work.

Three operators that a serving step runs one after the other:

  rotary     positions with one or three axes rotate the query and key heads of a batch of tokens
  append     a step's new keys (rotated by position) and values are quantized into the pages of a paged
             cache, and the step's queries are rotated on the way; pages hold TurboQuant blocks or 8-bit
             codes with one scale per 16 tokens and head
  attention  query tokens attend over 8-bit pages, causally: one token per sequence, a few drafted
             tokens, or a prompt

`own` false: elementary torch operations.  `own` true: the calls a program makes of leankv_b200.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

BLOCK = 16          # tokens that share one scale of an 8-bit page
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LEVELS = {
    2: [-1.0, -0.2997714, 0.2997714, 1.0],
    3: [-1.0, -0.6245203, -0.3513239, -0.1138989, 0.1138989, 0.3513239, 0.6245203, 1.0],
    4: [-1.0, -0.7573038, -0.5923403, -0.4599576, -0.3450764, -0.2405254, -0.1421261, -0.0470277,
        0.0470277, 0.1421261, 0.2405254, 0.3450764, 0.4599576, 0.5923403, 0.7573038, 1.0],
}
BORDERS = {
    2: [-0.6498857, 0.0, 0.6498857],
    3: [-0.8122602, -0.4879221, -0.2326114, 0.0, 0.2326114, 0.4879221, 0.8122602],
    4: [-0.8786519, -0.6748221, -0.5261490, -0.4025170, -0.2928009, -0.1913257, -0.0945769, 0.0,
        0.0945769, 0.1913257, 0.2928009, 0.4025170, 0.5261490, 0.6748221, 0.8786519],
}
BLOCK_BYTES = {2: 10, 3: 14, 4: 18}


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # one decode token of one sequence: the launch itself
        dict(name="rotary token", op="rotary", batch=1, tokens=1, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             axes=1, interleaved=False, inverse=False, dtype="bf16", far=100000),
        # an image-and-text prompt whose positions have three axes (time, height, width)
        dict(name="rotary prompt, three axes", op="rotary", batch=2, tokens=8192, q_heads=32, kv_heads=8, head_dim=128,
             rotary_dim=128, axes=3, interleaved=False, inverse=False, dtype="bf16", far=4000),
        # the gradient's direction, neighbouring pairs, a part of the head, an odd number of tokens
        dict(name="rotary gradient, part of the head", op="rotary", batch=3, tokens=1517, q_heads=16, kv_heads=2,
             head_dim=256, rotary_dim=64, axes=1, interleaved=True, inverse=True, dtype="f16", far=1000000),
        # a decode step of a full batch into TQ3 / TQ4 pages
        dict(name="append token, tq3 keys", op="append", bits=3, batch=64, tokens=1, q_heads=64, kv_heads=8,
             head_dim=128, page=16, axes=1, past=64, ragged=False, dtype="bf16"),
        # a long prompt into TQ4 pages, three position axes
        dict(name="append prompt, tq4 keys", op="append", bits=4, batch=1, tokens=16384, q_heads=32, kv_heads=8,
             head_dim=128, page=64, axes=3, past=0, ragged=False, dtype="bf16"),
        # a decode step into 8-bit pages: the touched blocks may have to be rescaled
        dict(name="append token, 8 bits", op="append", bits=8, batch=16, tokens=1, q_heads=32, kv_heads=8,
             head_dim=128, page=16, axes=1, past=64, ragged=False, dtype="bf16"),
        # a padded batch of prompt pieces behind what the cache holds, into 8-bit pages
        dict(name="append padded prompts, 8 bits", op="append", bits=8, batch=4, tokens=2000, q_heads=16, kv_heads=4,
             head_dim=256, page=32, axes=1, past=100, ragged=True, dtype="f16"),
        # one sequence, one token, a short context: latency
        dict(name="attention token, short", op="attention", batch=1, tokens=1, q_heads=32, kv_heads=8, head_dim=128,
             page=16, past=1000, ragged=False, dtype="bf16"),
        # a decode step over long contexts: the cache's bytes
        dict(name="attention token, long", op="attention", batch=16, tokens=1, q_heads=32, kv_heads=8, head_dim=128,
             page=64, past=32767, ragged=False, dtype="bf16"),
        # a few drafted tokens of each sequence, lengths of all kinds
        dict(name="attention drafted tokens", op="attention", batch=24, tokens=5, q_heads=64, kv_heads=8, head_dim=128,
             page=16, past=9000, ragged=True, dtype="bf16"),
        # a whole prompt
        dict(name="attention prompt", op="attention", batch=1, tokens=8192, q_heads=32, kv_heads=8, head_dim=128,
             page=128, past=0, ragged=False, dtype="bf16"),
        # padded prompt pieces behind cached prefixes, wide heads
        dict(name="attention prompt pieces", op="attention", batch=3, tokens=777, q_heads=16, kv_heads=4, head_dim=256,
             page=32, past=5000, ragged=True, dtype="f16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.499)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "attention", "attention"])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 8] if op != "attention" else [1, 3, 4, 8])
    wide = rng.random() < 0.3
    c = dict(op=op, q_heads=kv * group, kv_heads=kv, head_dim=256 if wide else 128, dtype=rng.choice(["bf16", "bf16", "f16"]))
    if op == "rotary":
        c["tokens"] = _spread(rng, 1, 8000)
        c["batch"] = _spread(rng, 1, max(1, min(64, 8000 // c["tokens"])))
        c["rotary_dim"] = rng.choice([c["head_dim"], c["head_dim"] // 2])
        c["axes"] = rng.choice([1, 3])
        c["interleaved"], c["inverse"] = rng.random() < 0.3, rng.random() < 0.3
        c["far"] = _spread(rng, 10, 1000000)
    elif op == "append":
        c["tokens"] = rng.choice([1, 1, _spread(rng, 2, 7000)])
        c["batch"] = _spread(rng, 1, max(1, min(64, 7000 // c["tokens"])))
        c["bits"] = rng.choice([2, 3, 4, 8, 8])
        c["page"] = rng.choice([16, 32, 64, 256])
        c["axes"] = rng.choice([1, 3])
        c["past"], c["ragged"] = rng.choice([0, _spread(rng, 1, 200)]), rng.random() < 0.5
    else:
        c["tokens"] = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 9, 4000)])
        most = int(1.3e11 / (c["tokens"] * c["q_heads"] * c["head_dim"])) - c["tokens"] // 2   # the listed prompt's work
        c["past"] = min(rng.choice([0, _spread(rng, 1, 16000)]), max(0, most))
        room = 16000 if c["tokens"] < 9 else 4000   # so that the scores of the plain form fit
        c["batch"] = _spread(rng, 1, max(1, min(16, room * 4 // (c["tokens"] * 4 + c["past"] + 1))))
        c["page"] = rng.choice([16, 32, 64, 256])
        c["ragged"] = rng.random() < 0.5
    return c


# ── inputs ───────────────────────────────────────────────────────────────────

def _channels(c, gen):
    """Key and value channels of unlike size, a few of them large, as projections give them."""
    s = torch.exp(0.4 * torch.randn(c["kv_heads"], c["head_dim"], generator=gen, device=DEV))
    s[:, :: c["head_dim"] // 4] *= 8.0
    return s


def _heads(c, gen):
    """Query, key and value heads [batch, heads, tokens, head_dim] as views of one projection's output."""
    b, n, hq, hk, d = c["batch"], c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    x = torch.randn(b, n, hq + 2 * hk, d, generator=gen, device=DEV)
    x[:, :, hq:hq + hk] *= _channels(c, gen)
    x = x.to(TYPES[c["dtype"]])
    return tuple(t.transpose(1, 2) for t in x.split([hq, hk, hk], dim=2))


def _positions(c, gen, first):
    """int32 [axes, batch, tokens]: text runs along all axes alike, an image's patches along height and width."""
    b, n = c["batch"], c["tokens"]
    i = torch.arange(n, device=DEV).expand(b, n)
    first = first.view(b, 1)
    if c["axes"] == 1:
        return (first + i).to(torch.int32)
    side = 1 + int(math.isqrt(max(1, n // 4)))
    patch = (i % (side * side + side)) < side * side
    time = first + i // (side * side + side)
    return torch.stack([time, torch.where(patch, first + (i % (side * side)) // side, first + i),
                        torch.where(patch, first + i % side, first + i)]).to(torch.int32).contiguous()


def _frequencies(c, dim):
    """Angle per position step and pair, and the axis that each pair turns with (sections as 1 : 1.5 : 1.5)."""
    pairs = dim // 2
    freq = 10000.0 ** (-2.0 * torch.arange(pairs, dtype=torch.float64) / dim)
    if c["axes"] == 1:
        return freq.to(DEV), None
    t, h = pairs // 4, 3 * pairs // 8
    axis = torch.tensor([0] * t + [1] * h + [2] * (pairs - t - h), dtype=torch.int32)
    return freq.to(DEV), axis.to(DEV)


def _table(c, most, gen):
    """int32 page table [batch, pages] over a shuffled pool, and the pool's number of pages."""
    per = -(-most // c["page"])
    total = c["batch"] * per
    order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    return order.view(c["batch"], per).contiguous(), total


def _lengths(c, gen):
    """Tokens that each sequence's cache holds before the step, and the step's tokens of each."""
    b = c["batch"]
    past = torch.full((b,), c["past"], dtype=torch.int32, device=DEV)
    new = torch.full((b,), c["tokens"], dtype=torch.int32, device=DEV)
    if c["past"] and (c["ragged"] or c["op"] == "append"):
        past = torch.randint(0, c["past"] + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
    if c["ragged"] and c["tokens"] > 1:
        new = torch.randint(1, c["tokens"] + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
    return past, new


def _blocks8(x):
    """8-bit codes and scales of rows [..., tokens, head_dim], tokens a multiple of 16."""
    y = x.unflatten(-2, (-1, BLOCK))
    s = y.abs().amax((-1, -2)) * (1.0 / 127.0)
    code = torch.round(y * (1.0 / s)[..., None, None]).clamp_(-127, 127).to(torch.int8)
    return code.flatten(-3, -2), s


def _pool8(c, table, total, gen, scaled):
    """Int8 pool [pages, kv_heads, page, head_dim] of Hadamard-rotated rows and its scales [pages, kv_heads, page / 16]."""
    h, p, d = c["kv_heads"], c["page"], c["head_dim"]
    code = torch.empty(total, h, p, d, dtype=torch.int8, device=DEV)
    scale = torch.empty(total, h, p // BLOCK, dtype=torch.float32, device=DEV)
    turn = _hadamard_matrix(d).float()
    for some in torch.arange(total, device=DEV).split(max(1, (1 << 26) // (h * p * d))):
        x = torch.randn(len(some), h, p, d, generator=gen, device=DEV)
        code[some], scale[some] = _blocks8((x * scaled[:, None] if scaled is not None else x) @ turn)
    return code, scale


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "rotary":
        s["q"], s["k"], _ = _heads(c, gen)
        first = torch.randint(0, c["far"], (c["batch"],), generator=gen, device=DEV)
        s["positions"] = _positions(c, gen, first)
        s["freq"], s["axis"] = _frequencies(c, c["rotary_dim"])
        return s
    past, new = _lengths(c, gen)
    s["table"], total = _table(c, c["past"] + c["tokens"], gen)
    s["pos"], s["new"], s["len"] = past, new, past + new
    s["max_len"] = c["past"] + c["tokens"]
    h, p, d = c["kv_heads"], c["page"], c["head_dim"]
    if c["op"] == "append":
        s["q"], s["k"], s["v"] = _heads(c, gen)
        s["freq"], s["axis"] = _frequencies(c, d)
        s["positions"] = None if c["axes"] == 1 else _positions(c, gen, past)
        if c["bits"] == 8:
            s["k_pool"], s["k_scale"] = _pool8(c, s["table"], total, gen, _channels(c, gen))
            s["v_pool"], s["v_scale"] = _pool8(c, s["table"], total, gen, None)
        else:
            s["k_pool"] = torch.zeros(total, h, p, d // 32, BLOCK_BYTES[c["bits"]], dtype=torch.uint8, device=DEV)
            s["v_pool"] = torch.zeros(total, h, p, d // 32, BLOCK_BYTES[4], dtype=torch.uint8, device=DEV)
    else:
        s["q"] = _heads(c, gen)[0]
        s["k_pool"], s["k_scale"] = _pool8(c, s["table"], total, gen, _channels(c, gen))
        s["v_pool"], s["v_scale"] = _pool8(c, s["table"], total, gen, None)
    return s


# ── plain forms ──────────────────────────────────────────────────────────────

def _stage(x, h):
    a = x.unflatten(-1, (-1, 2, h))
    u, w = a[..., 0, :], a[..., 1, :]
    return torch.stack((u + w, u - w), -2).flatten(-3)


def _hadamard(x):
    """The normalized Walsh-Hadamard transform of each row, the strides 1, 2, 4, ... in turn."""
    d = x.shape[-1]
    norm = (torch.ones(()) / torch.tensor(float(d)).sqrt()).item()
    return functools.reduce(_stage, [1 << i for i in range(d.bit_length() - 1)], x) * norm


def _turned(x, cos, sin, interleaved):
    """x [batch, heads, tokens, head_dim] in 32 bits with its leading pairs turned; cos, sin [batch, tokens, pairs]."""
    r = 2 * cos.shape[-1]
    x = x.float()
    c, s = cos[:, None], sin[:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    p, q = a * c - b * s, b * c + a * s
    head = torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1)
    return torch.cat((head, x[..., r:]), -1)


def _angles(positions, freq, axis, inverse=False):
    """cos and sin [batch, tokens, pairs] in 32 bits from 64-bit angles."""
    where = positions.double()[..., None] if axis is None else positions.double()[axis.long()].movedim(0, -1)
    angle = where * freq
    return angle.cos().float(), (-angle if inverse else angle).sin().float()


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s["positions"], s["freq"], s["axis"], c["inverse"])
    return tuple(_turned(s[t], cos, sin, c["interleaved"]).to(s[t].dtype) for t in ("q", "k"))


def _rows_of(s, bits, rows, pool, scale):
    """The pool's values after the rows [batch, kv_heads, tokens, head_dim] have been appended to it."""
    c = s["case"]
    h, p, d, n, b = c["kv_heads"], c["page"], c["head_dim"], c["tokens"], c["batch"]
    table, pos, new = s["table"].long(), s["pos"].long(), s["new"].long()
    t = torch.arange(n, device=DEV)
    slot = pos[:, None] + t
    fine = t < new[:, None]
    if bits != 8:
        y = rows.unflatten(-1, (-1, 32))
        top = y.abs().amax(-1, keepdim=True)
        inv = torch.where(top > 0, 1.0 / top, torch.zeros_like(top))
        code = torch.bucketize(y * inv, torch.tensor(BORDERS[bits], device=DEV))
        kept = (top.view(torch.int32) & -8192).view(torch.float32)   # the fp16 scale, truncated
        kept = torch.where(top < 2.0 ** -14, torch.zeros_like(kept), kept)
        value = (torch.tensor(LEVELS[bits], device=DEV)[code] * kept).flatten(-2)
        # padding goes to a page behind the pool
        page = torch.where(fine, table.gather(1, (slot // p).clamp(max=table.shape[1] - 1)), pool.shape[0])
        out = torch.zeros(pool.shape[0] + 1, h, p, d, dtype=torch.float32, device=DEV)
        out[page, :, slot % p] = value.transpose(1, 2)
        return out[:-1].to(s["k"].dtype)
    # 8 bits: the 16-token blocks that the rows touch, each with what it held before `pos`
    nb = (n + 2 * BLOCK - 2) // BLOCK
    block = (pos // BLOCK)[:, None] + torch.arange(nb, device=DEV)
    per = p // BLOCK
    at = table.gather(1, (block // per).clamp(max=table.shape[1] - 1)) * per + block % per
    at = torch.where(block * BLOCK < (pos + new)[:, None], at, pool.shape[0] * per)   # untouched: behind the pool
    lead = pos[:, None] % BLOCK
    # the row of each slot of those blocks; other slots take the zero row behind the last
    here = torch.arange(nb * BLOCK, device=DEV) - lead
    inside = (here >= 0) & (here < new[:, None])
    row = torch.where(inside, here, n)[:, None, :, None].expand(b, h, nb * BLOCK, d)
    x = torch.cat((rows, torch.zeros_like(rows[:, :, :1])), 2).gather(2, row)
    x = x.unflatten(2, (nb, BLOCK)).transpose(1, 2)                             # [b, nb, h, 16, d]
    codes = pool.unflatten(2, (per, BLOCK)).transpose(1, 2).flatten(0, 1)       # [pages * per, h, 16, d]
    scales = scale.transpose(1, 2).flatten(0, 1)                                # [pages * per, h]
    codes, scales = torch.cat((codes, codes[:1])), torch.cat((scales, scales[:1]))
    inside, older = (m.unflatten(1, (nb, BLOCK))[:, :, None, :, None] for m in (inside, here < 0))
    before = torch.where(older.any(3).squeeze(-1), scales[at], torch.zeros_like(scales[at]))
    s_new = torch.maximum(before, x.abs().amax((-1, -2)) * (1.0 / 127.0))
    inv = (1.0 / s_new)[..., None, None]
    fresh = torch.round(x * inv).clamp(-127, 127)
    held = codes[at].float()
    grown = torch.round(held * (before[..., None, None] * inv))
    moved = torch.where(inside, fresh, torch.where(older & (before < s_new)[..., None, None], grown, held))
    codes[at], scales[at] = moved.to(torch.int8), s_new
    value = codes[:-1].float() * scales[:-1, :, None, None]
    return value.unflatten(0, (-1, per)).transpose(1, 2).flatten(2, 3).to(s["k"].dtype)


def _plain_append(s):
    c = s["case"]
    b, n = c["batch"], c["tokens"]
    positions = s["positions"]
    if positions is None:
        positions = s["pos"][:, None] + torch.arange(n, device=DEV, dtype=torch.int32)
    cos, sin = _angles(positions, s["freq"], s["axis"])
    q = _turned(s["q"], cos, sin, False).to(s["q"].dtype)
    k = _rows_of(s, c["bits"], _hadamard(_turned(s["k"], cos, sin, False)), s["k_pool"], s.get("k_scale"))
    v = _rows_of(s, 8 if c["bits"] == 8 else 4, _hadamard(s["v"].float()), s["v_pool"], s.get("v_scale"))
    return q, k, v


def _pages(pool, scale, table):
    """Values [batch, kv_heads, tokens, head_dim] in 32 bits of an 8-bit pool's pages."""
    value = pool[table.long()].float().unflatten(3, (-1, BLOCK)) * scale[table.long()][..., None, None]
    return value.flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    c = s["case"]
    b, n, h, d = c["batch"], c["tokens"], c["kv_heads"], c["head_dim"]
    k, v = _pages(s["k_pool"], s["k_scale"], s["table"]), _pages(s["v_pool"], s["v_scale"], s["table"])
    q = _hadamard(s["q"].float()).unflatten(1, (h, -1)).flatten(2, 3)           # [b, h, group * n, d]
    score = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).unflatten(2, (-1, n))     # [b, h, group, n, tokens]
    i = torch.arange(n, device=DEV)
    last = (s["len"] - s["new"])[:, None] + i                                   # the last token that row i sees
    last = torch.where(i < s["new"][:, None], last, -1)
    seen = torch.arange(k.shape[2], device=DEV) <= last[..., None]              # [b, n, tokens]
    seen = seen[:, None, None]
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = score.sub_(top).exp_()
    out = p.flatten(2, 3) @ v / p.sum(-1, keepdim=True).clamp_(min=1e-30).flatten(2, 3)
    return _hadamard(out).unflatten(2, (-1, n)).flatten(1, 2).to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention}[c["op"]](s)
    from leankv_b200 import attention, ops
    if c["op"] == "rotary":
        rope = ops.Rotary(s["freq"], axis=s["axis"], interleaved=c["interleaved"])
        return ops.rotary(s["q"], s["positions"], rope, k=s["k"], inverse=c["inverse"])
    if c["op"] == "append":
        rope = ops.Rotary(s["freq"], axis=s["axis"])
        new = s["new"] if c["ragged"] else None
        q = ops.kv_append_rotary_paged(s["k"], s["v"], s["k_pool"], s["v_pool"], s["table"], s["pos"], rope=rope,
                                       positions=s["positions"], q=s["q"], new_len=new, k_scale=s.get("k_scale"),
                                       v_scale=s.get("v_scale"))
        kind = s["k"].dtype
        if c["bits"] == 8:
            return q, ops.dequantize_q8(s["k_pool"], s["k_scale"], kind), ops.dequantize_q8(s["v_pool"], s["v_scale"], kind)
        return q, ops.dequantize(s["k_pool"], c["bits"], kind), ops.dequantize(s["v_pool"], 4, kind)
    return attention.attention_q8_paged(s["q"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"],
                                        s["len"], q_len=s["new"] if c["ragged"] else None, max_kv_len=s["max_len"])


# ── work ─────────────────────────────────────────────────────────────────────

def work(case):
    c = case
    b, n, hq, hk, d = c["batch"], c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    size = 4 if c["dtype"] == "f32" else 2
    rows = b * n
    if c["op"] == "rotary":
        return {"bytes": 2 * rows * (hq + hk) * d * size + 4 * rows * c["axes"],
                "flops": 3 * rows * (hq + hk) * c["rotary_dim"]}
    filled = 0.5 if c["ragged"] and n > 1 else 1.0   # lengths are even between one and all tokens
    if c["op"] == "append":
        stored = 2 * d + 2 * 4 / BLOCK if c["bits"] == 8 else d // 32 * (BLOCK_BYTES[c["bits"]] + 18)
        pages = b * -(-(c["past"] + n) // c["page"])
        values = 2 * pages * c["page"] * hk * d
        moved = 2 * rows * hq * d * size + filled * rows * hk * (2 * d * size + stored)
        # the pool's values are returned: its codes are read and the values written
        return {"bytes": moved + values * size + values * (stored / (2 * d)),
                "flops": 3 * rows * hq * d + filled * rows * hk * d * (3 + 2 * (math.log2(d) + 8))}
    held = c["past"] * (0.5 if c["ragged"] else 1.0)
    tokens = b * (held + filled * n)
    seen = b * filled * n * (held + filled * n / 2)
    return {"bytes": tokens * hk * (2 * d + 2 * 4 / BLOCK) + 2 * rows * hq * d * size, "flops": 4 * seen * hq * d}


# ── exact values ─────────────────────────────────────────────────────────────

def _hadamard_matrix(d):
    """The symmetric orthogonal Hadamard matrix in 64 bits: entry (i, j) has the sign of the parity of i & j."""
    i = torch.arange(d, device=DEV)
    both = i[:, None] & i
    odd = torch.zeros_like(both)
    for bit in range(d.bit_length()):
        odd ^= (both >> bit) & 1
    return (1 - 2 * odd).double() / math.sqrt(d)


def _exact_turn(x, positions, freq, axis, interleaved, inverse):
    """Pairs as complex numbers, turned by exp(i angle)."""
    r = 2 * freq.numel()
    at = positions.double()
    angle = torch.stack([(at if axis is None else at[int(axis[j])]) * float(freq[j]) for j in range(r // 2)], -1)
    turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)[:, None]
    y = x.double().clone()
    even = list(range(0, r, 2)) if interleaved else list(range(r // 2))
    odd = [e + 1 for e in even] if interleaved else [e + r // 2 for e in even]
    z = torch.complex(y[..., even], y[..., odd]) * turn
    y[..., even], y[..., odd] = z.real, z.imag
    return y


def _exact_pool(s, bits, rows, pool, scale):
    c = s["case"]
    p = c["page"]
    if bits == 8:
        value = pool.double() * scale.double().repeat_interleave(BLOCK, -1)[..., None]
    else:
        value = torch.zeros(*pool.shape[:3], c["head_dim"], dtype=torch.float64, device=DEV)
    for b in range(c["batch"]):
        pos, end = int(s["pos"][b]), int(s["pos"][b] + s["new"][b])
        if bits != 8:
            y = rows[b, :, : end - pos].unflatten(-1, (-1, 32))
            top = y.abs().amax(-1, keepdim=True)
            code = torch.bucketize(y / top, torch.tensor(BORDERS[bits], device=DEV).double())
            step = torch.exp2(torch.floor(torch.log2(top)) - 10)     # the last bit that an fp16 scale keeps
            kept = torch.where(top < 2.0 ** -14, 0.0, torch.floor(top / step) * step)
            got = (torch.tensor(LEVELS[bits], device=DEV).double()[code] * kept).flatten(-2)
            slot = torch.arange(pos, end, device=DEV)
            value[s["table"][b].long()[slot // p], :, slot % p] = got.transpose(0, 1)
            continue
        for first in range(pos // BLOCK * BLOCK, end, BLOCK):
            page, off = int(s["table"][b, first // p]), first % p
            lo, hi = max(pos, first), min(end, first + BLOCK)
            y = rows[b, :, lo - pos: hi - pos]
            s_old = scale[page, :, off // BLOCK].double() if lo > first else torch.zeros(c["kv_heads"], device=DEV).double()
            s_new = torch.maximum(y.abs().amax((-1, -2)) / 127, s_old)
            at = value[page, :, off: off + BLOCK]
            codes = pool[page, :, off: off + BLOCK].double()
            grown = torch.where((s_old < s_new)[:, None, None], torch.round(codes * (s_old / s_new)[:, None, None]), codes)
            now = torch.arange(first, first + BLOCK, device=DEV)[None, :, None]
            # rows behind the appended ones keep their codes, under the block's new scale
            at[:] = torch.where(now < lo, grown, codes) * s_new[:, None, None]
            at[:, lo - first: hi - first] = torch.round(y / s_new[:, None, None]) * s_new[:, None, None]
    return value


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "rotary":
        return tuple(_exact_turn(s[t], s["positions"], s["freq"], s["axis"], c["interleaved"], c["inverse"]) for t in ("q", "k"))
    turn = _hadamard_matrix(c["head_dim"])
    if c["op"] == "append":
        if c["bits"] == 8 and c["batch"] * c["tokens"] > 20000:
            return None
        where = s["positions"]
        if where is None:
            where = s["pos"][:, None].double() + torch.arange(c["tokens"], device=DEV)
        q, k = (_exact_turn(s[t], where, s["freq"], s["axis"], False, False) for t in ("q", "k"))
        return q, _exact_pool(s, c["bits"], k @ turn, s["k_pool"], s.get("k_scale")), \
            _exact_pool(s, 8 if c["bits"] == 8 else 4, s["v"].double() @ turn, s["v_pool"], s.get("v_scale"))
    group = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(c["batch"]):
        total, new = int(s["len"][b]), int(s["new"][b])
        pages = s["table"][b].long()
        for h in range(c["kv_heads"]):
            k, v = ((s[t + "_pool"][pages, h].double() * s[t + "_scale"][pages, h].double().repeat_interleave(BLOCK, -1)[..., None])
                    .flatten(0, 1)[:total] for t in ("k", "v"))
            hide = torch.arange(total, device=DEV) > total - new + torch.arange(new, device=DEV)[:, None]
            for g in range(h * group, (h + 1) * group):
                w = s["q"][b, g, :new].double() @ turn @ k.T / math.sqrt(c["head_dim"])
                out[b, g, :new] = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ v @ turn
    return out
