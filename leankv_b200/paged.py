"""Paged TurboQuant KV cache for serving: sequences of independent lengths share page pools.

Every layer keeps a K pool and a V pool, uint8 [num_pages, n_kv_heads, page_size,
head_dim / 32, block_bytes] (TQ2_0, TQ3_0 or TQ4_0 keys, TQ4_0 values), or, with k_bits=8,
int8 [num_pages, n_kv_heads, page_size, head_dim] with one float32 scale per 16 tokens and
head: the tier that keeps prompts attendable, since its attention takes any number of query
tokens.  A page holds
page_size consecutive tokens of one sequence for every KV head; page p of sequence s
is pool page table[s, p], the same page in every layer's pools.  New rows are
Hadamard-rotated and quantized straight into their pages (tq_kv_append_paged_cuda)
and decode attention reads the pages in place (tq_decode_attention_paged_cuda): the
cache is never dequantized.  This is the paged form of the packed cache that
prototype/turboquant/kv_cache.py:109-204 keeps per layer.

A decode step:

    cache = PagedKVCache(n_layers, n_kv_heads=8, head_dim=128, num_pages=4096)
    a, b = cache.add_sequence(), cache.add_sequence()
    step = cache.batch([a, b], n_new=1)          # reserves pages, gathers the page rows
    for layer in range(n_layers):
        cache.append(step, layer, k, v)          # [2, n_kv_heads, 1, head_dim]
        out = cache.attention(step, layer, q)    # [2, n_q_heads, head_dim], sees the new rows
    cache.commit(step)                           # the sequences are one token longer
    cache.free_sequence(a)                       # its pages return to the pool

With a position rotation (ops.Rotary), append takes the keys as they leave the projection and
rotates keys and queries on the way, in the same launch:

    q = cache.append(step, layer, k, v, rope=rope, q=q)

With k_bits=8 a step may have any number of tokens, and sequences of different numbers of them
(new_len, a padded batch):

    step = cache.batch([a, b], n_new=[300, 25])  # rows 25 .. 299 of b are padding
    q = cache.append(step, layer, k, v, rope=rope, q=q)
    out = cache.attention(step, layer, q)        # [2, n_q_heads, 300, head_dim]

Drafted tokens of which some are rejected: instead of the drafts' step a batch of the accepted
counts is committed (their rows are in the pages already); later rows take the rejected ones'
slots.  8-bit blocks that held a rejected row keep a scale that is large enough for it.

    drafts = cache.batch([a, b], 5)
    ...                                          # append, attention, acceptance
    cache.commit(cache.batch([a, b], [2, 4]))

Page bookkeeping (PageTable) is host-side and needs no GPU.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Sequence

import numpy as np

NO_PAGE = -1   # page-table entry of a page not allocated (appends there are skipped and counted)


class PageTable:
    """Host-side page allocation: a free list of pool pages and one page-table row per sequence slot."""

    def __init__(self, num_pages: int, page_size: int, max_seqs: int, max_pages_per_seq: int):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two >= 16")
        if num_pages <= 0 or max_seqs <= 0 or max_pages_per_seq <= 0:
            raise ValueError("num_pages, max_seqs and max_pages_per_seq must be positive")
        self.num_pages, self.page_size = num_pages, page_size
        self.max_seqs, self.max_pages_per_seq = max_seqs, max_pages_per_seq
        self.table = np.full((max_seqs, max_pages_per_seq), NO_PAGE, dtype=np.int32)
        self.lens = np.zeros(max_seqs, dtype=np.int64)
        self.n_pages = np.zeros(max_seqs, dtype=np.int64)   # pages held per sequence
        self.active = np.zeros(max_seqs, dtype=bool)
        self._free = list(range(num_pages - 1, -1, -1))     # pop() hands out low pages first
        self.dirty: set = set()                             # sequence rows changed since the last sync

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def capacity(self) -> int:
        """Tokens one sequence can hold."""
        return self.max_pages_per_seq * self.page_size

    def add_sequence(self) -> int:
        idle = np.flatnonzero(~self.active)
        if idle.size == 0:
            raise RuntimeError(f"all {self.max_seqs} sequence slots are in use")
        s = int(idle[0])
        self.active[s] = True
        self.lens[s] = 0
        return s

    def free_sequence(self, s: int) -> None:
        self._check(s)
        held = self.table[s, : self.n_pages[s]]
        self._free.extend(int(p) for p in held[::-1])
        self.table[s, :] = NO_PAGE
        self.n_pages[s] = 0
        self.lens[s] = 0
        self.active[s] = False
        self.dirty.add(s)

    @staticmethod
    def _counts(seqs: Sequence[int], n_new) -> List[int]:
        """New tokens of each sequence: one number for all, or one each."""
        if isinstance(n_new, (list, tuple, np.ndarray)):
            counts = [int(n) for n in n_new]
            if len(counts) != len(seqs):
                raise ValueError("n_new must have one count per sequence")
        else:
            counts = [int(n_new)] * len(seqs)
        if any(n < 0 for n in counts):
            raise ValueError("token counts must not be negative")
        return counts

    def reserve(self, seqs: Sequence[int], n_new) -> None:
        """Give every sequence in seqs pages for n_new more tokens (one number, or one each; all or nothing)."""
        need = []
        for s, n in zip(seqs, self._counts(seqs, n_new)):
            self._check(s)
            total = int(self.lens[s]) + n
            if total > self.capacity:
                raise ValueError(f"sequence {s} would hold {total} tokens; the limit is {self.capacity}")
            need.append(max(0, -(-total // self.page_size) - int(self.n_pages[s])))
        if sum(need) > len(self._free):
            raise MemoryError(f"{sum(need)} pages needed, {len(self._free)} free")
        for s, n in zip(seqs, need):
            for _ in range(n):
                self.table[s, self.n_pages[s]] = self._free.pop()
                self.n_pages[s] += 1
            if n:
                self.dirty.add(s)

    def commit(self, seqs: Sequence[int], n_new) -> None:
        for s, n in zip(seqs, self._counts(seqs, n_new)):
            self._check(s)
            if self.lens[s] + n > self.n_pages[s] * self.page_size:
                raise ValueError(f"sequence {s}: {n} tokens were not reserved")
            self.lens[s] += n

    def _check(self, s: int) -> None:
        if not (0 <= s < self.max_seqs) or not self.active[s]:
            raise ValueError(f"sequence {s} is not active")


@dataclass
class Batch:
    """One step's sequences: their page-table rows, append positions and attention lengths (device)."""
    seqs: List[int]
    n_new: int           # rows of the step's tensors per sequence
    table: "object"      # int32 [B, max_pages_per_seq]
    pos: "object"        # int32 [B]: the first slot the step writes
    kv_len: "object"     # int32 [B]: pos + the sequence's new tokens
    max_kv_len: int
    counts: "object" = None    # new tokens of each sequence where they differ (else n_new each)
    new_len: "object" = None   # int32 [B]: the same on the device
    seen_len: "object" = None  # int32 [B]: kv_len, 0 where a sequence has only padding (None: none has)


class PagedKVCache:
    """Per-layer TurboQuant page pools with fused paged append and decode attention."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, num_pages: int, page_size: int = 16,
                 max_seqs: int = 64, max_pages_per_seq: int | None = None, k_bits: int = 3, k_opt_passes: int = 0,
                 device: str = "cuda"):
        import torch
        if head_dim not in (128, 256):
            raise ValueError("head_dim must be 128 or 256 (fused decode attention)")
        if k_bits not in (2, 3, 4, 8):
            raise ValueError("keys are TQ2_0, TQ3_0 or TQ4_0, or 8-bit codes (both pools)")
        if k_opt_passes and k_bits != 3:
            raise ValueError("optimal rounding applies to TQ3_0 keys")
        max_pages_per_seq = max_pages_per_seq or num_pages
        self.pages = PageTable(num_pages, page_size, max_seqs, max_pages_per_seq)
        self.n_layers, self.n_kv_heads, self.head_dim = n_layers, n_kv_heads, head_dim
        self.k_bits, self.k_opt_passes = k_bits, k_opt_passes
        self.device = torch.device(device)
        zeros = lambda shape, dtype: [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(n_layers)]   # noqa: E731
        if k_bits == 8:
            shape = (num_pages, n_kv_heads, page_size, head_dim)
            scales = (num_pages, n_kv_heads, page_size // 16)
            self.k, self.v = zeros(shape, torch.int8), zeros(shape, torch.int8)
            self.k_scale, self.v_scale = zeros(scales, torch.float32), zeros(scales, torch.float32)
        else:
            shape = (num_pages, n_kv_heads, page_size, head_dim // 32)
            self.k = zeros(shape + ({2: 10, 3: 14, 4: 18}[k_bits],), torch.uint8)
            self.v = zeros(shape + (18,), torch.uint8)
            self.k_scale = self.v_scale = [None] * n_layers
        self._table = torch.full((max_seqs, max_pages_per_seq), NO_PAGE, dtype=torch.int32, device=self.device)
        self._lens = torch.zeros(max_seqs, dtype=torch.int32, device=self.device)

    # sequence management (host bookkeeping; page-table rows reach the device in batch())
    def add_sequence(self) -> int:
        s = self.pages.add_sequence()
        self._lens[s] = 0
        return s

    def free_sequence(self, s: int) -> None:
        self.pages.free_sequence(s)

    def seq_len(self, s: int) -> int:
        return int(self.pages.lens[s])

    def batch(self, seqs: Sequence[int], n_new=1) -> Batch:
        """Reserve pages for n_new tokens of every sequence and gather the step's device views.  With a count
        for each sequence the step's tensors have max(n_new) rows, those behind a sequence's count are padding."""
        import torch
        seqs = [int(s) for s in seqs]
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence may appear once per batch")
        counts = self.pages._counts(seqs, n_new)
        self.pages.reserve(seqs, counts)
        self._sync()
        idx = torch.tensor(seqs, dtype=torch.int64, device=self.device)
        pos = self._lens.index_select(0, idx)
        lens = self.pages.lens[seqs] + np.asarray(counts, dtype=np.int64)
        rows = max(counts, default=0)
        alike = all(n == rows for n in counts)
        new_len = None if alike else torch.tensor(counts, dtype=torch.int32, device=self.device)
        kv_len = (pos + (rows if alike else new_len)).contiguous()
        return Batch(seqs, rows, self._table.index_select(0, idx).contiguous(), pos.contiguous(), kv_len,
                     int(lens.max()) if len(seqs) else 0, None if alike else counts, new_len,
                     None if alike or min(counts) else kv_len * (new_len > 0))

    def append(self, step: Batch, layer: int, k, v, rope=None, positions=None, q=None):
        """Quantize-on-write of the step's new rows k, v [B, n_kv_heads, n_new, head_dim].

        rope (ops.Rotary): k (and q [B, n_q_heads, n_new, head_dim], whose rotated rows are returned) as they
        leave the projection, any strides; turned by their positions (default: their slots; int32 [B, n_new]
        or [axes, B, n_new] otherwise) in the same launch."""
        import torch
        from . import ops
        B = len(step.seqs)
        for t, name in ((k, "k"), (v, "v")):
            if tuple(t.shape) != (B, self.n_kv_heads, step.n_new, self.head_dim):
                raise ValueError(f"{name} must be [{B}, {self.n_kv_heads}, {step.n_new}, {self.head_dim}]")
        if q is not None and rope is None:
            raise ValueError("q is taken for its rotation: give rope")
        if self.k_opt_passes == 0 and (rope is not None or self.k_bits == 8 or step.new_len is not None):
            return ops.kv_append_rotary_paged(k, v, self.k[layer], self.v[layer], step.table, step.pos, rope=rope,
                                              positions=positions, q=q, new_len=step.new_len,
                                              k_scale=self.k_scale[layer], v_scale=self.v_scale[layer])
        if step.new_len is not None:
            raise ValueError("optimal rounding takes batches without padding")
        out = None
        if rope is not None:
            # optimal rounding is a pass of its own: the keys are rotated in float32 before it
            where = positions if positions is not None else \
                (step.pos[:, None] + torch.arange(step.n_new, dtype=torch.int32, device=self.device)).contiguous()
            out = ops.rotary(q, where, rope) if q is not None else None
            k = ops.rotary(k.float(), where, rope)
        ops.kv_append_paged(k.contiguous(), self.k[layer], step.table, step.pos, qtype=self.k_bits,
                            opt_passes=self.k_opt_passes)
        ops.kv_append_paged(v.contiguous(), self.v[layer], step.table, step.pos, qtype=4)
        return out

    def attention(self, step: Batch, layer: int, q, sm_scale: float | None = None, out_dtype=None, out=None):
        """Attention over each sequence's tokens, this step's included: q [B, n_q_heads, head_dim], one token per
        sequence (its last), or, with k_bits=8, [B, n_q_heads, n_new, head_dim], each row seeing the tokens up to its
        own; rows of padding, in the first form those of sequences without a token in a step of unequal counts, give
        zeros.  attention.last_status() tells whether a kernel met a page id outside the pool or gave up a wait."""
        from . import attention as A
        if self.k_bits == 8:
            if q.dim() == 4 and q.shape[2] != step.n_new:
                raise ValueError(f"q must have the step's {step.n_new} tokens")
            # one row per sequence out of several is the last one: a count above q's rows is taken as their number
            return A.attention_q8_paged(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                        step.table, step.kv_len, q_len=step.new_len,
                                        max_kv_len=step.max_kv_len, sm_scale=sm_scale, out_dtype=out_dtype or q.dtype, out=out)
        lens = step.kv_len if step.seen_len is None else step.seen_len
        return A.decode_attention_paged(q.contiguous(), self.k[layer], self.v[layer], step.table, lens,
                                        max_kv_len=step.max_kv_len, sm_scale=sm_scale,
                                        out_dtype=out_dtype or q.dtype, out=out)

    def commit(self, step: Batch) -> None:
        """The step's rows are part of the sequences from now on."""
        import torch
        self.pages.commit(step.seqs, step.n_new if step.counts is None else step.counts)
        idx = torch.tensor(step.seqs, dtype=torch.int64, device=self.device)
        self._lens.index_copy_(0, idx, step.kv_len)

    def _sync(self) -> None:
        import torch
        if not self.pages.dirty:
            return
        rows = sorted(self.pages.dirty)
        self.pages.dirty.clear()
        idx = torch.tensor(rows, dtype=torch.int64, device=self.device)
        self._table.index_copy_(0, idx, torch.from_numpy(self.pages.table[rows]).to(self.device))
        for s in rows:
            if not self.pages.active[s]:
                self._lens[s] = 0

    def memory_summary(self) -> dict:
        pool = sum(t.numel() for t in self.k) + sum(t.numel() for t in self.v)
        pool += sum(4 * t.numel() for t in self.k_scale + self.v_scale if t is not None)
        used = self.pages.num_pages - self.pages.free_pages
        return {"pool_bytes": pool, "pages": self.pages.num_pages, "pages_used": used,
                "page_size": self.pages.page_size, "bytes_per_page_all_layers": pool // self.pages.num_pages,
                "tokens_cached": int(self.pages.lens[self.pages.active].sum())}
