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

A tree of drafted tokens (k_bits=8): its nodes are appended like a step's tokens, rotated by their depths, and see the
cached tokens and their ancestors; the accepted path's rows then move up behind the cached ones.  A step
rounds the rows of the block of 16 slots that it begins in up to twice more, when a node raises the block's scale and when the
path's move sets it back: the rows that stay are off by about 1.4 times what a chain of the same tokens leaves (200 steps of
26 nodes and 4 accepted, rows of unlike size: 2.4e-2 of the norm, the chain 1.6e-2).

    step = cache.batch([a, b], n, tree=parents)  # parents of the n nodes, -1 for children of the cached tokens
    q = cache.append(step, layer, k, v, rope=rope, q=q)
    out = cache.attention(step, layer, q)
    cache.accept(step, [[0, 2, 5], [1]])         # in place of the commit

Eviction (track_weights=True): attention counts the weights that cached tokens get, evict drops those with the least of
them, each KV head of each layer its own; positions go on counting from the tokens that a sequence has had.

    out = cache.attention(step, layer, q, observe=1)   # the last query token of each sequence counts
    cache.evict([a, b], keep=1024, sinks=4, recent=128)

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
        self.dropped = np.zeros(max_seqs, dtype=np.int64)   # tokens evicted: what positions are ahead of slots
        self.n_pages = np.zeros(max_seqs, dtype=np.int64)   # pages held per sequence
        self.active = np.zeros(max_seqs, dtype=bool)
        self.given_back = np.zeros(max_seqs, dtype=np.int64)   # how often a sequence slot has given tokens or pages back
        self.times_given_back = 0                              # all slots together
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
        self.dropped[s] = 0
        return s

    def free_sequence(self, s: int) -> None:
        self._check(s)
        held = self.table[s, : self.n_pages[s]]
        self._free.extend(int(p) for p in held[::-1])
        self.table[s, :] = NO_PAGE
        self.n_pages[s] = 0
        self.lens[s] = 0
        self.dropped[s] = 0
        self.active[s] = False
        self._gives_back(s)
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

    def truncate(self, s: int, length: int) -> None:
        """The sequence keeps its first `length` tokens; pages behind them return to the pool."""
        self._check(s)
        if not 0 <= length <= self.lens[s]:
            raise ValueError(f"sequence {s} has {int(self.lens[s])} tokens")
        held = -(-length // self.page_size)
        self._free.extend(int(p) for p in self.table[s, held: self.n_pages[s]][::-1])
        if held < self.n_pages[s] or length < self.lens[s]:
            self._gives_back(s)
        if held < self.n_pages[s]:
            self.table[s, held: self.n_pages[s]] = NO_PAGE
            self.n_pages[s] = held
            self.dirty.add(s)
        self.dropped[s] += self.lens[s] - length
        self.lens[s] = length

    def _gives_back(self, s: int) -> None:
        self.given_back[s] += 1
        self.times_given_back += 1

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
    positions: "object" = None # int32 [B, n_new] where they are not the slots (trees, sequences with evicted tokens)
    tree: "object" = None      # ops.DraftTree
    parents: "object" = None   # the tree's, numpy [B or 1, n_new] (None: they came from the device)
    starts: "object" = None    # pos and kv_len on the host
    ends: "object" = None
    index: "object" = None     # seqs as an array
    given_back: "object" = None      # the sequences' PageTable.given_back when the step was made
    times_given_back: "object" = None
    written: "object" = None         # layers whose rows have been appended (caches that track weights)


class PagedKVCache:
    """Per-layer TurboQuant page pools with fused paged append and decode attention."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, num_pages: int, page_size: int = 16,
                 max_seqs: int = 64, max_pages_per_seq: int | None = None, k_bits: int = 3, k_opt_passes: int = 0,
                 device: str = "cuda", track_weights: bool = False):
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
        # sums of attention weights beside the pages, every layer's
        self._weights = torch.zeros((n_layers, num_pages, n_kv_heads, page_size), dtype=torch.float32, device=self.device) \
            if track_weights else None
        self.weights = [None] * n_layers if self._weights is None else list(self._weights)
        # Drafted tokens may be observed and rejected.  Of each sequence: the slots behind its tokens that may hold weights end at
        # _observed; in a layer, the weights from _valid on are of rows that others have been written over.
        self._observed = np.zeros(max_seqs, dtype=np.int64)
        self._valid = np.zeros((n_layers, max_seqs), dtype=np.int64)

    # sequence management (host bookkeeping; page-table rows reach the device in batch())
    def add_sequence(self) -> int:
        s = self.pages.add_sequence()
        self._lens[s] = 0
        self._observed[s] = 0
        self._valid[:, s] = 0
        return s

    def free_sequence(self, s: int) -> None:
        self.pages.free_sequence(s)

    def seq_len(self, s: int) -> int:
        return int(self.pages.lens[s])

    def batch(self, seqs: Sequence[int], n_new=1, tree=None) -> Batch:
        """Reserve pages for n_new tokens of every sequence and gather the step's device views.  With a count
        for each sequence the step's tensors have max(n_new) rows, those behind a sequence's count are padding.

        tree: the tokens are nodes of trees of drafted tokens: their parents, which come before them (-1: the cached
        tokens), [max(n_new)] for all sequences or [B, max(n_new)], from the host or an int32 CUDA tensor."""
        import torch
        seqs = [int(s) for s in seqs]
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence may appear once per batch")
        for s in seqs:
            self.pages._check(s)
        counts = self.pages._counts(seqs, n_new)
        rows = max(counts, default=0)
        parents = None
        if tree is not None:
            if self.k_bits != 8:
                raise ValueError("trees are attended in 8-bit pages (k_bits=8)")
            if not isinstance(tree, torch.Tensor) or not tree.is_cuda:
                parents = np.atleast_2d(np.asarray(tree, dtype=np.int32))
                if parents.ndim != 2 or (parents >= np.arange(parents.shape[1])).any() or (parents < -1).any():
                    raise ValueError("parents must come before their nodes, -1 for children of the cached tokens")
                tree = torch.from_numpy(parents).to(self.device)
            if tuple(tree.shape) not in ((rows,), (1, rows), (len(seqs), rows)):
                raise ValueError(f"tree must have the step's {rows} nodes, one tree or {len(seqs)} of them")
        fresh_pages = self.pages.n_pages[seqs].copy() if self._weights is not None else None
        self.pages.reserve(seqs, counts)
        if fresh_pages is not None:
            got = [int(p) for s, n in zip(seqs, fresh_pages) for p in self.pages.table[s, n: self.pages.n_pages[s]]]
            if got:
                self._weights.index_fill_(1, torch.tensor(got, dtype=torch.int64, device=self.device), 0.0)
        self._sync()
        idx = torch.tensor(seqs, dtype=torch.int64, device=self.device)
        pos = self._lens.index_select(0, idx)
        index = np.asarray(seqs, dtype=np.int64)
        lens = self.pages.lens[index] + np.asarray(counts, dtype=np.int64)
        alike = all(n == rows for n in counts)
        new_len = None if alike else torch.tensor(counts, dtype=torch.int32, device=self.device)
        kv_len = (pos + (rows if alike else new_len)).contiguous()
        step = Batch(seqs, rows, self._table.index_select(0, idx).contiguous(), pos.contiguous(), kv_len,
                     int(lens.max()) if len(seqs) else 0, None if alike else counts, new_len,
                     None if alike or min(counts) else kv_len * (new_len > 0), parents=parents,
                     starts=self.pages.lens[index], ends=lens, index=index, given_back=self.pages.given_back[index],
                     times_given_back=self.pages.times_given_back)
        dropped = self.pages.dropped[seqs]
        if tree is not None or dropped.any():
            from . import ops
            first = pos + torch.from_numpy(dropped.astype(np.int32)).to(self.device)
            ahead = torch.arange(rows, dtype=torch.int32, device=self.device)
            if tree is not None:
                step.tree = ops.draft_tree(tree)
                ahead = step.tree.depth
            step.positions = (first[:, None] + ahead).contiguous()
        return step

    def append(self, step: Batch, layer: int, k, v, rope=None, positions=None, q=None):
        """Quantize-on-write of the step's new rows k, v [B, n_kv_heads, n_new, head_dim].

        rope (ops.Rotary): k (and q [B, n_q_heads, n_new, head_dim], whose rotated rows are returned) as they
        leave the projection, any strides; turned by their positions (default: the tokens that came before, a tree's
        nodes by their depths; int32 [B, n_new] or [axes, B, n_new] otherwise) in the same launch."""
        import torch
        from . import ops
        self._check_step(step)
        if self._weights is not None and step.starts is not None:
            if not step.written or layer in step.written:   # once for all layers, and again when the step's rows are written anew
                self._valid[:, step.index] = np.minimum(self._valid[:, step.index], step.starts)
                step.written = set()
            step.written.add(layer)
        B = len(step.seqs)
        if positions is None and rope is not None:
            positions = step.positions
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

    def attention(self, step: Batch, layer: int, q, sm_scale: float | None = None, out_dtype=None, out=None,
                  return_lse: bool = False, observe: int = 0, decay: float = 1.0):
        """Attention over each sequence's tokens, this step's included: q [B, n_q_heads, head_dim], one token per
        sequence (its last), or, with k_bits=8, [B, n_q_heads, n_new, head_dim], each row seeing the tokens up to its
        own (a tree's node: its ancestors); rows of padding, in the first form those of sequences without a token in a step of
        unequal counts, give zeros.  attention.last_status() tells whether a kernel met a page id outside the pool or gave up a wait.

        observe: that many of each sequence's last query tokens count towards the weights by which evict() chooses, earlier
        counts times decay (track_weights=True; after a tree's step the accepted rows count by observe())."""
        from . import attention as A
        self._check_step(step)
        if observe and step.tree is not None:
            raise ValueError("nodes of a tree may be rejected: observe() the accepted ones after accept()")
        if observe:
            self._need_weights()
        want_lse = return_lse or bool(observe)
        if self.k_bits == 8:
            if q.dim() == 4 and q.shape[2] != step.n_new:
                raise ValueError(f"q must have the step's {step.n_new} tokens")
            if step.tree is not None and q.dim() == 3 and step.n_new != 1:
                raise ValueError(f"q must have the step's {step.n_new} nodes")
            # one row per sequence out of several is the last one: a count above q's rows is taken as their number
            got = A.attention_q8_paged(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                       step.table, step.kv_len, q_len=step.new_len, max_kv_len=step.max_kv_len,
                                       sm_scale=sm_scale, out_dtype=out_dtype or q.dtype, out=out, return_lse=want_lse,
                                       tree=step.tree)
        else:
            lens = step.kv_len if step.seen_len is None else step.seen_len
            got = A.decode_attention_paged(q.contiguous(), self.k[layer], self.v[layer], step.table, lens,
                                           max_kv_len=step.max_kv_len, sm_scale=sm_scale,
                                           out_dtype=out_dtype or q.dtype, out=out, return_lse=want_lse)
        if observe:
            self.observe(step, layer, q, got[1], window=int(observe), decay=decay, sm_scale=sm_scale)
        return got if return_lse or not want_lse else got[0]

    def observe(self, step: Batch, layer: int, q, lse, window: int | None = None, decay: float = 1.0,
                sm_scale: float | None = None) -> None:
        """Counts the attention weights of the step's query rows (the last `window` of each sequence, default all), whose
        attention left lse, towards the weights by which evict() chooses; earlier counts times decay.  Once a step and layer:
        the step's own tokens begin at nothing.  After accept(), with the step it returns and the rows of q and lse of the
        accepted nodes, as the rows of a chain."""
        from . import attention as A
        self._check_step(step)
        self._need_weights()
        if step.tree is not None:
            raise ValueError("nodes of a tree may be rejected: observe the accepted ones after accept()")
        lens = step.kv_len if step.seen_len is None else step.seen_len
        A.attention_weights_paged(q, self.k[layer], step.table, lens, lse, self.weights[layer], k_scale=self.k_scale[layer],
                                  q_len=step.new_len, fresh=step.pos, decay=decay, window=window,
                                  max_kv_len=step.max_kv_len, sm_scale=sm_scale)
        self._observed[step.index] = np.maximum(self._observed[step.index], step.ends)
        self._valid[layer, step.index] = step.ends

    def accept(self, step: Batch, nodes: Sequence[Sequence[int]]) -> Batch:
        """In place of the commit of a tree's step: of each sequence the nodes of a path (rising, none for a sequence that
        accepts nothing) become its next tokens, the others are forgotten.  Returns the step of the accepted rows, committed."""
        import torch
        from . import ops
        if step.tree is None:
            raise ValueError("the step has no tree")
        paths = [[int(x) for x in p] for p in nodes]
        if len(paths) != len(step.seqs):
            raise ValueError("nodes must have one path per sequence")
        for i, path in enumerate(paths):
            limit = step.n_new if step.counts is None else step.counts[i]
            before = [-1] + path
            if any(not a < x < limit for a, x in zip(before, path)):
                raise ValueError(f"sequence {step.seqs[i]}: a path rises within its {limit} nodes")
            if step.parents is not None:
                row = step.parents[i if len(step.parents) > 1 else 0]
                if any(int(row[x]) != a for a, x in zip(before, path)):
                    raise ValueError(f"sequence {step.seqs[i]}: {path} is not a path of the tree")
        self._check_step(step)
        for s, n in zip(step.seqs, step.starts):
            if n != self.pages.lens[s]:
                raise ValueError(f"sequence {s} has changed since the step")
        rows = max((len(p) for p in paths), default=0)
        if rows:
            src = torch.tensor([p + [-1 << 30] * (rows - len(p)) for p in paths], dtype=torch.int32, device=self.device)
            src = src + step.pos[:, None]
            for layer in range(self.n_layers):
                ops.kv_move_paged(self.k[layer], self.v[layer], step.table, src, first=step.pos, k_scale=self.k_scale[layer],
                                  v_scale=self.v_scale[layer])
        kept = self.batch(step.seqs, [len(p) for p in paths])
        self.commit(kept)
        return kept

    def evict(self, seqs: Sequence[int], keep, sinks: int = 0, recent: int = 0) -> None:
        """Drops tokens of the sequences until `keep` (one number, or one each) are left: in every layer each KV head keeps its
        last `recent` and first `sinks` tokens and, of the others, those with the largest observed weights.  Pages that are
        no longer needed return to the pool; later tokens' positions are not changed by it.  Steps made before an eviction are
        refused from then on where it took tokens from one of their sequences."""
        import torch
        from . import ops
        self._need_weights()
        seqs = [int(s) for s in seqs]
        many = self.pages._counts(seqs, keep)
        step = self.batch(seqs, 0)
        left = [min(n, int(self.pages.lens[s])) for s, n in zip(seqs, many)]
        width = max((n for s, n in zip(seqs, left) if n < self.pages.lens[s]), default=0)
        if all(n == self.pages.lens[s] for s, n in zip(seqs, left)):
            return
        count = torch.tensor(left, dtype=torch.int32, device=self.device)
        # sequences that keep all their tokens have nothing to move
        moved = torch.tensor([n if n < self.pages.lens[s] else 0 for s, n in zip(seqs, left)], dtype=torch.int32, device=self.device)
        for layer in range(self.n_layers if width else 0):
            slots = ops.select_tokens(self.weights[layer], step.table, step.kv_len, moved, sinks=sinks, recent=recent,
                                      width=width, max_kv_len=step.max_kv_len)
            ops.kv_move_paged(self.k[layer], self.v[layer], step.table, slots, k_scale=self.k_scale[layer],
                              v_scale=self.v_scale[layer], weights=self.weights[layer])
        # (the others keep what a step under way has reserved and observed)
        cut = [(s, n) for s, n in zip(seqs, left) if n < self.pages.lens[s]]
        for s, n in cut:
            self._observed[s] = self.pages.capacity
            self.pages.truncate(s, n)
        self._forget([s for s, _ in cut], [n for _, n in cut])
        self._lens.index_copy_(0, torch.tensor(seqs, dtype=torch.int64, device=self.device), count)

    def _forget(self, seqs: Sequence[int], starts: Sequence[int]) -> None:
        """Slots behind the sequences' tokens begin at nothing (pages that join a sequence do anyway), and so do those from
        starts on whose weights are of other rows than they hold."""
        import torch
        size, t = self.pages.page_size, self.pages
        lengths, tops = t.lens[seqs], np.minimum(self._observed[seqs], t.n_pages[seqs] * size)
        firsts = np.clip(self._valid[:, seqs], starts, lengths)
        tails: dict = {}   # layers (None: all) -> (page, slot) of each
        for i in np.flatnonzero((firsts < tops).any(0)):
            for first in np.unique(firsts[:, i]):
                here = firsts[:, i] == first
                layers = None if here.all() else tuple(np.flatnonzero(here))
                tails.setdefault(layers, []).extend((int(t.table[seqs[i], x // size]), x % size) for x in range(int(first), int(tops[i])))
        self._observed[seqs] = np.minimum(self._observed[seqs], lengths)
        self._valid[:, seqs] = np.minimum(self._valid[:, seqs], lengths)
        for layers, tail in tails.items():
            if tail:
                page, slot = (torch.tensor(i, dtype=torch.int64, device=self.device) for i in zip(*tail))
                for weights in [self._weights] if layers is None else [self._weights[n: n + 1] for n in layers]:
                    weights[:, page, :, slot] = 0.0

    def _check_step(self, step: Batch) -> None:
        """A step has its own copy of page-table rows: of a sequence that has been freed or evicted from they name pages that
        others may hold by now."""
        if step.times_given_back == self.pages.times_given_back or step.given_back is None:
            return
        if (self.pages.given_back[step.index] != step.given_back).any():
            raise ValueError("a sequence has been freed or evicted from since the step was made: its slots and pages are no longer those of "
                             "the step")

    def _need_weights(self) -> None:
        if self._weights is None:
            raise ValueError("weights are not tracked: PagedKVCache(track_weights=True)")

    def commit(self, step: Batch) -> None:
        """The step's rows are part of the sequences from now on."""
        if step.tree is not None:
            raise ValueError("a tree's step is committed by accept()")
        self._check_step(step)
        import torch
        starts = [int(n) for n in self.pages.lens[step.seqs]]
        self.pages.commit(step.seqs, step.n_new if step.counts is None else step.counts)
        idx = torch.tensor(step.seqs, dtype=torch.int64, device=self.device)
        self._lens.index_copy_(0, idx, step.kv_len)
        if self._weights is not None:
            self._forget(step.seqs, starts)

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
        pool += sum(4 * t.numel() for t in self.k_scale + self.v_scale + self.weights if t is not None)
        used = self.pages.num_pages - self.pages.free_pages
        return {"pool_bytes": pool, "pages": self.pages.num_pages, "pages_used": used,
                "page_size": self.pages.page_size, "bytes_per_page_all_layers": pool // self.pages.num_pages,
                "tokens_cached": int(self.pages.lens[self.pages.active].sum())}
