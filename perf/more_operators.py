"""Cases of four operators of a paged cache that drafts trees and evicts tokens: inputs, plain forms, exact values, work.

  tree     the nodes of a tree of drafted tokens attend over 8-bit pages, each to the cached tokens and its ancestors
  weights  the attention weights that cached tokens got from a step's queries are added up, over 8-bit or TurboQuant keys
  select   the tokens of each sequence and KV head that stay: the first, the last and those of the most weight
  move     rows of the pages are moved together: the accepted path of a tree, or the tokens that stay

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
        # a small tree behind a short context: latency
        dict(name="tree, one sequence", op="tree", batch=1, tokens=10, q_heads=32, kv_heads=8, head_dim=128, page=16,
             past=1000, ragged=False, dtype="bf16"),
        # a verification step of a full batch, lengths and trees of all sizes
        dict(name="tree, batch", op="tree", batch=16, tokens=26, q_heads=32, kv_heads=8, head_dim=128, page=64,
             past=9000, ragged=True, dtype="bf16"),
        # wide trees, wide heads, many query heads to a KV head
        dict(name="tree, wide", op="tree", batch=3, tokens=63, q_heads=64, kv_heads=8, head_dim=256, page=32,
             past=12000, ragged=False, dtype="f16"),
        # a decode step that keeps account of the weights: one sequence, a short context
        dict(name="weights, one sequence", op="weights", bits=8, batch=1, tokens=1, q_heads=32, kv_heads=8, head_dim=128,
             page=16, past=1000, ragged=False, window=0, decay=1.0, dtype="bf16"),
        # the same over long contexts: the keys' bytes
        dict(name="weights, long", op="weights", bits=8, batch=16, tokens=1, q_heads=32, kv_heads=8, head_dim=128, page=64,
             past=32767, ragged=False, window=0, decay=0.98, dtype="bf16"),
        # the last queries of prompts vote on the prompts' tokens
        dict(name="weights, prompt's end", op="weights", bits=8, batch=2, tokens=100, q_heads=32, kv_heads=8, head_dim=128,
             page=128, past=16000, ragged=False, window=64, decay=0.0, dtype="bf16"),
        # a decode step over TQ3 keys, lengths of all kinds
        dict(name="weights, tq3 keys", op="weights", bits=3, batch=32, tokens=1, q_heads=64, kv_heads=8, head_dim=128, page=16,
             past=9000, ragged=True, window=0, decay=1.0, dtype="bf16"),
        # a short cache is cut to a quarter
        dict(name="select, one sequence", op="select", batch=1, kv_heads=8, page=16, past=1025, keep=256, sinks=4, recent=32,
             ragged=False),
        # long caches of a full batch
        dict(name="select, long", op="select", batch=16, kv_heads=8, page=64, past=32768, keep=8192, sinks=4, recent=128,
             ragged=False),
        # the accepted path of a tree moves up behind the cached tokens
        dict(name="move, accepted path", op="move", bits=8, batch=16, kv_heads=8, head_dim=128, page=16, past=64, tokens=26,
             keep=6, accept=True, ragged=True, weights=False, dtype="bf16"),
        # the tokens that stay move to the front of a full batch's long caches, and their weights with them
        dict(name="move, kept tokens", op="move", bits=8, batch=16, kv_heads=8, head_dim=128, page=64, past=32768, tokens=0,
             keep=8192, accept=False, ragged=False, weights=True, dtype="bf16"),
        # the same in TQ3 / TQ4 pages, wide heads, odd lengths
        dict(name="move, tq3 keys", op="move", bits=3, batch=5, kv_heads=4, head_dim=256, page=32, past=10001, tokens=0,
             keep=3001, accept=False, ragged=True, weights=False, dtype="f16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.499)))))))


def draw(rng):
    op = rng.choice(["tree", "weights", "weights", "select", "move"])
    c = dict(op=op, batch=_spread(rng, 1, 16), kv_heads=rng.choice([1, 2, 4, 8]), page=rng.choice([16, 32, 64, 256]),
             ragged=rng.random() < 0.5)
    if op in ("tree", "weights"):
        c["bits"] = 8 if op == "tree" else rng.choice([8, 8, 8, 2, 3, 4])
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 3, 4, 8])
        c["head_dim"] = rng.choice([128, 128, 256])
        c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
        if op == "tree":
            c["tokens"] = _spread(rng, 1, 100)
        else:
            c["tokens"] = rng.choice([1, rng.randint(2, 8), _spread(rng, 9, 200)]) if c["bits"] == 8 else 1
            c["window"] = rng.choice([0, 0, _spread(rng, 1, 64)])
            c["decay"] = rng.choice([1.0, 0.9, 0.0])
        # the scores of the plain form and the listed cases' work are the bounds
        rows = c["batch"] * c["q_heads"] * c["tokens"]
        c["past"] = rng.choice([0, _spread(rng, 1, max(1, min(16000, int(2.4e8 / rows), int(2.4e10 / (rows * c["head_dim"])))))])
    elif op == "select":
        c["past"] = _spread(rng, 1, 32000)
        c["keep"] = _spread(rng, 1, c["past"])
        c["sinks"], c["recent"] = rng.choice([0, 4]), rng.choice([0, _spread(rng, 1, 256)])
    else:
        c["bits"] = rng.choice([8, 8, 2, 3, 4])
        c["head_dim"] = rng.choice([128, 128, 256])
        c["accept"] = rng.random() < 0.4
        c["weights"], c["dtype"] = rng.random() < 0.5, rng.choice(["bf16", "f16"])
        c["past"] = _spread(rng, 1, 200 if c["accept"] else 16000)
        c["tokens"] = _spread(rng, 2, 100) if c["accept"] else 0
        c["keep"] = _spread(rng, 1, min(12, c["tokens"]) if c["accept"] else max(1, c["past"] // 2))
    return c


# ── inputs ───────────────────────────────────────────────────────────────────

def _channels(c, gen):
    """Key channels of unlike size, a few of them large, as projections give them."""
    s = torch.exp(0.4 * torch.randn(c["kv_heads"], c["head_dim"], generator=gen, device=DEV))
    s[:, :: c["head_dim"] // 4] *= 8.0
    return s


def _rows(c, gen, scaled, pages):
    """Head rows [pages, kv_heads, page, head_dim] as the pages hold them: Hadamard-rotated."""
    x = torch.randn(pages, c["kv_heads"], c["page"], c["head_dim"], generator=gen, device=DEV)
    return (x * scaled[:, None] if scaled is not None else x) @ _hadamard_matrix(c["head_dim"]).float()


def _pool8(c, total, gen, scaled):
    """Int8 pool [pages, kv_heads, page, head_dim] and its scales [pages, kv_heads, page / 16]."""
    h, p, d = c["kv_heads"], c["page"], c["head_dim"]
    code = torch.empty(total, h, p, d, dtype=torch.int8, device=DEV)
    scale = torch.empty(total, h, p // BLOCK, dtype=torch.float32, device=DEV)
    for some in torch.arange(total, device=DEV).split(max(1, (1 << 26) // (h * p * d))):
        y = _rows(c, gen, scaled, len(some)).unflatten(-2, (-1, BLOCK))
        s = y.abs().amax((-1, -2)) * (1.0 / 127.0)
        code[some] = torch.round(y * (1.0 / s)[..., None, None]).clamp_(-127, 127).to(torch.int8).flatten(-3, -2)
        scale[some] = s
    return code, scale


def _packed(code, bits):
    """Bytes [..., 4 * bits] of 32 codes."""
    if bits == 4:
        return code[..., :16] | code[..., 16:] << 4
    if bits == 2:
        return (code.unflatten(-1, (8, 4)) << torch.tensor([0, 2, 4, 6], device=DEV)).sum(-1)
    word = (code.unflatten(-1, (4, 8)) << 3 * torch.arange(8, device=DEV)).sum(-1)
    return (word[..., None] >> torch.tensor([0, 8, 16], device=DEV) & 255).flatten(-2)


def _pool_tq(c, bits, total, gen, scaled):
    """TurboQuant blocks uint8 [pages, kv_heads, page, head_dim / 32, bytes]."""
    h, p, d = c["kv_heads"], c["page"], c["head_dim"]
    pool = torch.empty(total, h, p, d // 32, BLOCK_BYTES[bits], dtype=torch.uint8, device=DEV)
    for some in torch.arange(total, device=DEV).split(max(1, (1 << 24) // (h * p * d))):
        y = _rows(c, gen, scaled, len(some)).unflatten(-1, (-1, 32))
        top = y.abs().amax(-1, keepdim=True)
        pool[some, ..., 2:] = _packed(torch.bucketize(y / top, torch.tensor(BORDERS[bits], device=DEV)), bits).to(torch.uint8)
        kept = (top.view(torch.int32) & -8192).view(torch.float32).half()     # the fp16 scale, truncated
        pool[some, ..., :2] = kept.view(torch.uint8)
    return pool


def _lengths(c, gen):
    """Tokens that each sequence's cache holds before the step, and the step's tokens of each."""
    b = c["batch"]
    past = torch.full((b,), c["past"], dtype=torch.int32, device=DEV)
    new = torch.full((b,), c.get("tokens", 0), dtype=torch.int32, device=DEV)
    if c["ragged"]:
        past = torch.randint(0, c["past"] + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
        if c.get("tokens", 0) > 1:
            new = torch.randint(1, c["tokens"] + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
    return past, new


def _tree(c, gen):
    """Ancestor masks of random trees whose later nodes hang from the likeliest earlier ones: truth values
    [batch, tokens, tokens], and the same as bits of int32 words [batch, tokens, ceil(tokens / 32)]."""
    b, n = c["batch"], c["tokens"]
    i = torch.arange(n, device=DEV)
    parent = (torch.rand(b, n, generator=gen, device=DEV).square() * (i + 1)).long().clamp(max=i) - 1   # -1: the cached tokens
    eye = torch.eye(n, dtype=torch.float32, device=DEV)
    step = eye + (parent[..., None] == i).float()
    seen = functools.reduce(lambda x, _: (x @ x).clamp_(max=1.0), range(n.bit_length()), step) > 0
    words = torch.nn.functional.pad(seen, (0, -n % 32)).unflatten(-1, (-1, 32)).long() << torch.arange(32, device=DEV)
    return seen, words.sum(-1).to(torch.int32).contiguous()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    b, h, p = c["batch"], c["kv_heads"], c["page"]
    past, new = _lengths(c, gen)
    s["pos"], s["new"], s["len"] = past, new, past + new
    s["max_len"] = c["past"] + c.get("tokens", 0)
    per = max(1, -(-s["max_len"] // p))
    total = b * per
    # pages in any order, but those that kept tokens will fill in front of the others
    front = per if c["op"] != "move" or c["accept"] else min(per, -(-c["keep"] // p))
    s["front"] = b * front
    first = torch.randperm(b * front, generator=gen, device=DEV).view(b, front)
    rest = b * front + torch.randperm(total - b * front, generator=gen, device=DEV).view(b, per - front)
    s["table"] = torch.cat((first, rest), 1).to(torch.int32).contiguous()
    if c["op"] in ("tree", "weights"):
        d, n, hq = c["head_dim"], c["tokens"], c["q_heads"]
        x = torch.randn(b, n, hq + 2 * h, d, generator=gen, device=DEV).to(TYPES[c["dtype"]])
        s["q"] = x[:, :, :hq].transpose(1, 2)     # a view of the projection's output
        scaled = _channels(c, gen)
        if c.get("bits", 8) != 8:
            s["k_pool"], s["k_scale"] = _pool_tq(c, c["bits"], total, gen, scaled), None
        else:
            s["k_pool"], s["k_scale"] = _pool8(c, total, gen, scaled)
    if c["op"] == "tree":
        s["v_pool"], s["v_scale"] = _pool8(c, total, gen, None)
        s["seen"], s["mask"] = _tree(c, gen)
    if c["op"] == "weights":
        s["lse"] = _lse(s)
        s["weights"] = _past_weights(total, h, p, gen)
        s["fresh"] = past
    if c["op"] == "select":
        s["weights"] = _past_weights(total, h, p, gen)
        s["keep"] = torch.full((b,), c["keep"], dtype=torch.int32, device=DEV)
        if c["ragged"]:
            s["keep"] = torch.randint(1, c["keep"] + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
    if c["op"] == "move":
        if c["bits"] == 8:
            s["k_pool"], s["k_scale"] = _pool8(c, total, gen, _channels(c, gen))
            s["v_pool"], s["v_scale"] = _pool8(c, total, gen, None)
        else:
            s["k_pool"], s["v_pool"] = _pool_tq(c, c["bits"], total, gen, _channels(c, gen)), _pool_tq(c, 4, total, gen, None)
            s["k_scale"] = s["v_scale"] = None
        s["weights"] = _past_weights(total, h, p, gen) if c["weights"] else None
        s["first"], s["src"] = _moves(s, gen)
    return s


def _past_weights(total, h, p, gen):
    """Weights that tokens have got so far: most of them little, some none, and many alike."""
    w = torch.exp(2.0 * torch.randn(total, h, p, generator=gen, device=DEV) - 6.0)
    kind = torch.rand(total, h, p, generator=gen, device=DEV)
    return torch.where(kind < 0.1, 0.0, torch.where(kind < 0.3, torch.round(w * 512) / 512, w))


def _moves(s, gen):
    """Slots that move and where the first of them goes: rising, -1 behind the last.  An accepted path is the same for all
    heads and lies among the step's slots, kept tokens are each head's own."""
    c = s["case"]
    b, h, m = c["batch"], c["kv_heads"], c["keep"]
    if c["accept"]:
        many = torch.minimum(s["new"], torch.randint(1, m + 1, (b,), generator=gen, device=DEV, dtype=torch.int32))
        u = torch.rand(b, c["tokens"], generator=gen, device=DEV)
        u[torch.arange(c["tokens"], device=DEV) >= s["new"][:, None]] = 2.0
        lead, shape = s["pos"][:, None], (b, m)
    else:
        many = torch.clamp(s["len"], max=m)
        u = torch.rand(b, h, c["past"], generator=gen, device=DEV)
        u.masked_fill_((torch.arange(c["past"], device=DEV) >= s["len"][:, None])[:, None], 2.0)
        lead, shape = 0, (b, h, m)
    many = many.view(b, *[1] * (len(shape) - 1))
    order = u.argsort(-1)[..., :m]
    none = torch.arange(order.shape[-1], device=DEV) >= many
    slots = order.masked_fill(none, 1 << 30).sort(-1).values + lead
    slots = torch.where(none, -1, slots).to(torch.int32)
    return (s["pos"] if c["accept"] else torch.zeros_like(s["pos"])), slots.contiguous()


def _lse(s):
    """The log-sum-exp that the step's attention has left for every query row, float32 [batch, q_heads, tokens]."""
    c = s["case"]
    out = []
    for b in range(c["batch"]):
        k = _keys(s, s["table"][b:b + 1])[0]
        q = _hadamard(s["q"][b].float()).unflatten(0, (c["kv_heads"], -1))
        score = (q.flatten(1, 2) @ k.transpose(-1, -2)).mul_(c["head_dim"] ** -0.5).unflatten(1, q.shape[1:3])
        score.masked_fill_(~_seen(s, k.shape[1])[b], -math.inf)
        out.append(score.logsumexp(-1).flatten(0, 1))
    return torch.stack(out)


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


def _unpacked(blocks, bits):
    """Values [..., head_dim] of TurboQuant blocks [..., head_dim / 32, bytes]."""
    by = blocks[..., 2:].int()
    if bits == 4:
        code = torch.cat((by & 15, by >> 4), -1)
    elif bits == 2:
        code = (by[..., None] >> torch.tensor([0, 2, 4, 6], device=DEV) & 3).flatten(-2)
    else:
        word = (by.unflatten(-1, (4, 3)) << torch.tensor([0, 8, 16], device=DEV)).sum(-1)
        code = (word[..., None] >> 3 * torch.arange(8, device=DEV) & 7).flatten(-2)
    d = blocks[..., :2].contiguous().view(torch.float16).float()
    return (torch.tensor(LEVELS[bits], device=DEV)[code] * d).flatten(-2)


def _pages(pool, scale, table):
    """Values [batch, kv_heads, tokens, head_dim] in 32 bits of an 8-bit pool's pages."""
    value = pool[table.long()].float().unflatten(3, (-1, BLOCK)) * scale[table.long()][..., None, None]
    return value.flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _keys(s, table):
    """Key values [batch, kv_heads, tokens, head_dim] in 32 bits."""
    if s["k_scale"] is not None:
        return _pages(s["k_pool"], s["k_scale"], table)
    return _unpacked(s["k_pool"][table.long()], s["case"]["bits"]).transpose(1, 2).flatten(2, 3)


def _seen(s, slots):
    """Truth values [batch, tokens, slots]: row i of a sequence sees the tokens up to its own."""
    i = torch.arange(s["case"]["tokens"], device=DEV)
    last = torch.where(i < s["new"][:, None], s["pos"][:, None] + i, -1)
    return torch.arange(slots, device=DEV) <= last[..., None]


def _seen_of_tree(s, slots):
    """The same for trees: the cached tokens, and the step's tokens that the mask has."""
    n = s["case"]["tokens"]
    slot = torch.arange(slots, device=DEV)
    node = slot - s["pos"][:, None]                                             # [batch, slots]
    among = (node >= 0) & (node < s["new"][:, None])
    at = node.clamp(0, n - 1)[:, None].expand(-1, n, -1)
    seen = (node < 0)[:, None] | (s["seen"].gather(2, at) & among[:, None])
    return seen & (torch.arange(n, device=DEV) < s["new"][:, None])[..., None]


def _plain_tree(s):
    c = s["case"]
    n, h, d = c["tokens"], c["kv_heads"], c["head_dim"]
    k, v = _pages(s["k_pool"], s["k_scale"], s["table"]), _pages(s["v_pool"], s["v_scale"], s["table"])
    q = _hadamard(s["q"].float()).unflatten(1, (h, -1)).flatten(2, 3)           # [b, h, group * n, d]
    score = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).unflatten(2, (-1, n))     # [b, h, group, n, tokens]
    score.masked_fill_(~_seen_of_tree(s, k.shape[2])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = score.sub_(top).exp_()
    out = p.flatten(2, 3) @ v / p.sum(-1, keepdim=True).clamp_(min=1e-30).flatten(2, 3)
    return _hadamard(out).unflatten(2, (-1, n)).flatten(1, 2).to(s["q"].dtype)


def _plain_weights(s):
    c = s["case"]
    n, h, d, p = c["tokens"], c["kv_heads"], c["head_dim"], c["page"]
    k = _keys(s, s["table"])
    q = _hadamard(s["q"].float()).unflatten(1, (h, -1)).flatten(2, 3)
    score = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).unflatten(2, (-1, n))
    seen = _seen(s, k.shape[2])
    if c["window"]:
        seen &= (torch.arange(n, device=DEV) >= s["new"][:, None] - c["window"])[..., None]
    e = score.sub_(s["lse"].unflatten(1, (h, -1))[..., None]).exp_().masked_fill_(~seen[:, None, None], 0.0)
    got = e.sum((2, 3))                                                         # [b, h, tokens]
    slot = torch.arange(k.shape[2], device=DEV)
    held = s["weights"][s["table"].long()].transpose(1, 2).flatten(2, 3)
    kept = torch.where((slot < s["fresh"][:, None])[:, None], held * c["decay"], 0.0)
    now = torch.where((slot < s["len"][:, None])[:, None], kept + got, held)
    s["weights"][s["table"].long()] = now.unflatten(2, (-1, p)).transpose(1, 2)
    return s["weights"]


def _plain_select(s):
    c = s["case"]
    w = s["weights"][s["table"].long()].transpose(1, 2).flatten(2, 3)           # [b, h, slots]
    slot = torch.arange(w.shape[2], device=DEV)
    length, k = s["len"][:, None, None], torch.minimum(s["keep"], s["len"])[:, None, None]
    recent = k.clamp(max=c["recent"])
    sinks = torch.minimum(k - recent, torch.full_like(k, c["sinks"]))
    rank = torch.where((slot >= length - recent) | (slot < sinks), 2.0 ** 100, w)
    rank = torch.where(slot < length, rank, -1.0)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    none = torch.arange(order.shape[-1], device=DEV) >= k
    slots = order.masked_fill(none, 1 << 30).sort(-1).values
    return torch.where(none, -1, slots).to(torch.int32)


def _rows_at(s, slots):
    """Rows of the pool, seen as [pages * kv_heads * page], of slots [batch, kv_heads, rows]."""
    h, p = s["case"]["kv_heads"], s["case"]["page"]
    page = s["table"].long().gather(1, (slots // p).flatten(1)).view_as(slots)
    return (page * h + torch.arange(h, device=DEV)[:, None]) * p + slots % p


def _plain_move(s):
    c = s["case"]
    b, h, p, d = c["batch"], c["kv_heads"], c["page"], c["head_dim"]
    src = s["src"].long() if s["src"].dim() == 3 else s["src"].long()[:, None].expand(-1, h, -1)
    lead = s["first"].long() % BLOCK                                            # older rows of the first block
    blocks = -(-(src.shape[2] + (BLOCK - 1 if c["accept"] else 0)) // BLOCK)
    j = torch.arange(blocks * BLOCK, device=DEV) - lead[:, None]                # [b, rows of whole blocks]
    to = (s["first"].long()[:, None] + j)[:, None].expand(b, h, -1)
    moved = torch.cat((src, torch.full_like(src[..., :1], -1)), 2).gather(
        2, torch.where((j >= 0) & (j < src.shape[2]), j, src.shape[2])[:, None].expand(b, h, -1))
    older = (j < 0)[:, None].expand_as(to)
    real = (moved >= 0) | older
    inside = to < s["table"].shape[1] * p
    to_row = _rows_at(s, torch.where(inside, to, 0))
    from_row = _rows_at(s, torch.where(moved >= 0, moved, torch.where(inside, to, 0)))
    kind = TYPES[c["dtype"]]
    w = None if s["weights"] is None else s["weights"].view(-1)
    if w is not None:
        w[to_row[inside]] = w[from_row][inside]
        w = s["weights"][:s["front"]]
    out = []
    for pool, scale, bits in ((s["k_pool"], s["k_scale"], c["bits"]), (s["v_pool"], s["v_scale"], 8 if c["bits"] == 8 else 4)):
        if bits != 8:
            rows = pool.view(-1, pool.shape[3] * pool.shape[4])
            rows[to_row[inside]] = rows[from_row][inside]
            out.append(_unpacked(pool[:s["front"]], bits).to(kind))
            continue
        codes, scales = pool.view(-1, d), scale.view(-1)
        held = codes[from_row].float()                                          # [b, h, rows, d]
        size = scales[from_row // BLOCK]
        top = held.abs().amax(-1) * size * (1.0 / 127.0)
        size, top, use = (x.unflatten(2, (-1, BLOCK)) for x in (size, top, real))
        most, least = size.masked_fill(~use, 0.0).amax(-1), size.masked_fill(~use, math.inf).amin(-1)
        now = torch.where(most == least, most, top.masked_fill(~use, 0.0).amax(-1))
        ratio = torch.where((now > 0)[..., None], size / now[..., None], 0.0).flatten(2)
        fresh = torch.round(held * ratio[..., None]).clamp_(-127, 127)
        codes[to_row[inside]] = torch.where(real[..., None], fresh, held).to(torch.int8)[inside]
        at, some = to_row.unflatten(2, (-1, BLOCK))[..., 0] // BLOCK, use.any(-1)
        scales[at[some]] = now[some]
        out.append((pool[:s["front"]].float().unflatten(2, (-1, BLOCK)) * scale[:s["front"]][..., None, None]).flatten(2, 3).to(kind))
    return out if w is None else out + [w]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"tree": _plain_tree, "weights": _plain_weights, "select": _plain_select, "move": _plain_move}[c["op"]](s)
    from leankv_b200 import attention, ops
    if c["op"] == "tree":
        return attention.attention_q8_paged(s["q"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"], s["len"],
                                            q_len=s["new"] if c["ragged"] else None, max_kv_len=s["max_len"], tree=s["mask"])
    if c["op"] == "weights":
        return attention.attention_weights_paged(s["q"], s["k_pool"], s["table"], s["len"], s["lse"], s["weights"],
                                                 k_scale=s["k_scale"], q_len=s["new"] if c["ragged"] else None, fresh=s["fresh"],
                                                 decay=c["decay"], window=c["window"] or None, max_kv_len=s["max_len"])
    if c["op"] == "select":
        return ops.select_tokens(s["weights"], s["table"], s["len"], s["keep"], sinks=c["sinks"], recent=c["recent"],
                                 width=c["keep"], max_kv_len=s["max_len"])
    ops.kv_move_paged(s["k_pool"], s["v_pool"], s["table"], s["src"], first=s["first"], k_scale=s["k_scale"],
                      v_scale=s["v_scale"], weights=s["weights"])
    kind, n = TYPES[c["dtype"]], s["front"]
    if c["bits"] == 8:
        out = [ops.dequantize_q8(s[t + "_pool"][:n], s[t + "_scale"][:n], kind) for t in ("k", "v")]
    else:
        out = [ops.dequantize(s["k_pool"][:n], c["bits"], kind), ops.dequantize(s["v_pool"][:n], 4, kind)]
    return out if s["weights"] is None else out + [s["weights"][:n]]


# ── work ─────────────────────────────────────────────────────────────────────

def work(case):
    c = case
    b, hk = c["batch"], c["kv_heads"]
    half = 0.5 if c["ragged"] else 1.0   # lengths are even between none or one and all tokens
    held = c["past"] * half
    if c["op"] in ("tree", "weights"):
        n, hq, d = c["tokens"], c["q_heads"], c["head_dim"]
        rows = n * (half if n > 1 else 1.0)
        tokens = b * (held + rows)
        key = d + 4 / BLOCK if c.get("bits", 8) == 8 else d // 32 * BLOCK_BYTES[c["bits"]]
        if c["op"] == "tree":
            return {"bytes": tokens * hk * 2 * key + 2 * b * n * hq * d * 2, "flops": 4 * b * rows * (held + rows / 4) * hq * d}
        rows = min(rows, c["window"]) if c["window"] else rows
        held_weights = 8 if c["decay"] else 4
        return {"bytes": tokens * hk * (key + held_weights) + b * rows * hq * (2 * d + 4),
                "flops": 2 * b * rows * (held + n / 2) * hq * d}
    if c["op"] == "select":
        kept = c["keep"] * half if c["keep"] > 1 else 1
        return {"bytes": 4 * b * hk * (held + kept), "flops": b * hk * held}
    d = c["head_dim"]
    rows = b * hk * (c["keep"] * (0.5 if c["accept"] else 1.0) if c["accept"] else min(c["keep"], held))
    stored = 2 * d + 2 * 4 / BLOCK if c["bits"] == 8 else d // 32 * (BLOCK_BYTES[c["bits"]] + 18)
    pages = b * (-(-(c["past"] + c["tokens"]) // c["page"]) if c["accept"] else -(-c["keep"] // c["page"]))
    values = 2 * pages * c["page"] * hk * d
    # the values of the pages that rows moved to are returned: their codes are read and the values written
    return {"bytes": rows * (2 * stored + 4 + (8 if c["weights"] else 0)) + values * 2 + values * stored / (2 * d),
            "flops": 4 * rows * 2 * d}


# ── exact values ─────────────────────────────────────────────────────────────

def _hadamard_matrix(d):
    """The symmetric orthogonal Hadamard matrix in 64 bits: entry (i, j) has the sign of the parity of i & j."""
    i = torch.arange(d, device=DEV)
    both = i[:, None] & i
    odd = torch.zeros_like(both)
    for bit in range(d.bit_length()):
        odd ^= (both >> bit) & 1
    return (1 - 2 * odd).double() / math.sqrt(d)


def _exact_blocks(blocks, bits):
    """Values of TurboQuant blocks in 64 bits: codes as a stream of bits, the lowest first; 4-bit codes lie in the order
    0, 16, 1, 17, ...; the scale's exponent and fraction are taken apart."""
    stream = (blocks[..., 2:, None].int() >> torch.arange(8, device=DEV) & 1).flatten(-2).unflatten(-1, (32, bits))
    code = (stream << torch.arange(bits, device=DEV)).sum(-1)
    code = torch.cat((code[..., 0::2], code[..., 1::2]), -1) if bits == 4 else code
    half = blocks[..., 0:1].long() + 256 * blocks[..., 1:2].long()
    size = (1024 + half % 1024).double() * torch.exp2((half // 1024 - 25).double())
    return (torch.tensor(LEVELS[bits], device=DEV).double()[code] * size).flatten(-2)


def _exact_rows(s, b, h, total, name="k"):
    """The first rows of one sequence and head, in 64 bits."""
    pages = s["table"][b].long()
    got = s[name + "_pool"][pages, h]
    if s[name + "_scale"] is None:
        return _exact_blocks(got, s["case"]["bits"] if name == "k" else 4).flatten(0, 1)[:total]
    return (got.double() * s[name + "_scale"][pages, h].double().repeat_interleave(BLOCK, -1)[..., None]).flatten(0, 1)[:total]


def _exact_tree(s):
    c = s["case"]
    turn, group = _hadamard_matrix(c["head_dim"]), c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(c["batch"]):
        past, new = int(s["pos"][b]), int(s["new"][b])
        hide = torch.cat((torch.zeros(new, past, dtype=torch.bool, device=DEV), ~s["seen"][b, :new, :new]), 1)
        for h in range(c["kv_heads"]):
            k, v = (_exact_rows(s, b, h, past + new, t) for t in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                w = s["q"][b, g, :new].double() @ turn @ k.T / math.sqrt(c["head_dim"])
                out[b, g, :new] = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ v @ turn
    return out


def _exact_weights(s):
    c = s["case"]
    turn, group, p = _hadamard_matrix(c["head_dim"]), c["q_heads"] // c["kv_heads"], c["page"]
    out = s["weights"].double()
    for b in range(c["batch"]):
        past, new = int(s["pos"][b]), int(s["new"][b])
        rows = torch.arange(max(0, new - c["window"]) if c["window"] else 0, new, device=DEV)
        slot = torch.arange(past + new, device=DEV)
        page = s["table"][b].long()[slot // p]
        for h in range(c["kv_heads"]):
            k = _exact_rows(s, b, h, past + new)
            held = out[page, h, slot % p] * c["decay"]
            held[int(s["fresh"][b]):] = 0
            for g in range(h * group, (h + 1) * group):
                w = s["q"][b, g, rows].double() @ turn @ k.T / math.sqrt(c["head_dim"])
                e = torch.exp(w - s["lse"][b, g, rows].double()[:, None])
                held += torch.where(slot <= past + rows[:, None], e, 0.0).sum(0)
            out[page, h, slot % p] = held
    return out


def _exact_select(s):
    """Each token's place by counting: how many come before it in the order of weight, then slot."""
    c = s["case"]
    out = torch.full((c["batch"], c["kv_heads"], c["keep"]), -1, dtype=torch.int32, device=DEV)
    for b in range(c["batch"]):
        n = int(s["len"][b])
        k = min(n, int(s["keep"][b]))
        recent = min(k, c["recent"])
        sinks = min(k - recent, c["sinks"])
        for h in range(c["kv_heads"]):
            w = s["weights"][s["table"][b].long(), h].flatten()[sinks: n - recent].double()
            some = k - recent - sinks
            border = torch.sort(w, descending=True).values[some - 1] if some else math.inf
            over = w > border
            ties = torch.nonzero(w == border).flatten()[: some - int(over.sum())] if some else torch.zeros(0, dtype=torch.long, device=DEV)
            kept = torch.cat((torch.arange(sinks, device=DEV), sinks + torch.nonzero(over).flatten(), sinks + ties,
                              torch.arange(n - recent, n, device=DEV)))
            out[b, h, :k] = kept.sort().values.to(torch.int32)
    return out


def _exact_move(s):
    c = s["case"]
    h, p, d, n = c["kv_heads"], c["page"], c["head_dim"], s["front"]
    wide = 8 if c["bits"] == 8 else 0
    w = None if s["weights"] is None else s["weights"].double()
    k, v = ((s[t + "_pool"].double() * s[t + "_scale"].double().repeat_interleave(BLOCK, -1)[..., None])[:n] if wide
            else _exact_blocks(s[t + "_pool"][:n], c["bits"] if t == "k" else 4) for t in ("k", "v"))
    heads = torch.arange(h, device=DEV)[:, None]
    for b in range(c["batch"]):
        first, table = int(s["first"][b]), s["table"][b].long()
        src = s["src"][b].long().view(-1, s["src"].shape[-1]).expand(h, -1)
        src = src[:, : int((src[0] >= 0).sum())]
        many = src.shape[1]
        if not many:
            continue
        to = torch.arange(first, first + many, device=DEV)
        if w is not None:
            w[table[to // p], :, to % p] = w[table[src // p], heads, src % p].T
        older = torch.arange(first // BLOCK * BLOCK, first, device=DEV)
        every = torch.cat((older, to))
        where = torch.cat((older.expand(h, -1), src), 1)
        for out, name in ((k, "k"), (v, "v")):
            pool, scale = s[name + "_pool"], s[name + "_scale"]
            if not wide:
                got = _exact_blocks(pool[table[where // p], heads, where % p], c["bits"] if name == "k" else 4)
                out[table[every // p], :, every % p] = got.transpose(0, 1)
                continue
            code = pool[table[where // p], heads, where % p].double()
            size = scale[table[where // p], heads, where % p // BLOCK].double()
            last = -(-(first + many) // BLOCK) * BLOCK
            behind = torch.arange(first + many, last, device=DEV)                # these keep their codes
            fill = (0, len(behind))
            top = torch.nn.functional.pad(code.abs().amax(-1) * size / 127, fill).unflatten(1, (-1, BLOCK)).amax(-1)
            most = torch.nn.functional.pad(size, fill).unflatten(1, (-1, BLOCK)).amax(-1)
            least = torch.nn.functional.pad(size, fill, value=math.inf).unflatten(1, (-1, BLOCK)).amin(-1)
            now = torch.where(most == least, most, top).repeat_interleave(BLOCK, 1)
            fresh = torch.round(code * (size / now[:, : len(every)])[..., None]) * now[:, : len(every), None]
            out[table[every // p], :, every % p] = fresh.transpose(0, 1)
            if len(behind):
                old = pool[table[behind // p], :, behind % p].double()
                out[table[behind // p], :, behind % p] = old * now[:, len(every):].T[..., None]
    return [k, v] if w is None else [k, v, w[:n]]


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "weights": _exact_weights, "select": _exact_select, "move": _exact_move}[case["op"]](s)
