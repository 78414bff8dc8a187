"""A multi-tenant decoder on the engine's operators: what a model says of
given tokens, every token under its own tenant's adapters.

`TenantDecoder` is a stack of pre-norm decoder layers whose projections run on
`engine.linear` (the gated MLP's two projections and their product in one
launch, residuals added in the epilogue), whose heads are normed and turned by
their positions on `engine.rotate_heads` where the model does that, whose
attention runs on `engine.packed_attention` over the packed prompts, and whose
logits are read once by `engine.token_logprobs`.  The adapters' deltas are
`engine.add_lora_packed` calls on the step's one segment table.

  * `score(ids, cu_seqlens, tenants)`: per token the log probability of the one
    after it -- scoring prompts, or the first step of a request (it leaves the
    prompts' keys and values in a `PackedCache`);
  * `verify(ids, cu_seqlens, tenants, cache)`: the same for tokens drafted after
    what the cache holds, all in one pass; the cache grows by them.

Both also take a `PagedCache`, whose rows stay where they were written
(`engine.rotate_into_cache`, `engine.paged_attention`): growing it copies
nothing, its sequences come and go, drafts are taken back by `cut`, and its rows
may be e4m3 of half the bytes.

Nothing here waits for the device; the lengths that the caller passes, and
where the cache's rows go, are uploaded from host memory at each step.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from .engine import TokenLogprobs, WarpPipeEngine
from .rotary import Rotary


class DecoderLayer(NamedTuple):
    """Weights of one layer; adapters as [K, 1, rank, in] and [K, 1, out, rank]
    or None.  w_gate_up holds the gate's rows, then the up projection's."""

    norm1: torch.Tensor
    w_qkv: torch.Tensor
    w_o: torch.Tensor
    norm2: torch.Tensor
    w_gate_up: torch.Tensor
    w_down: torch.Tensor
    qkv_a: Optional[torch.Tensor] = None
    qkv_b: Optional[torch.Tensor] = None
    o_a: Optional[torch.Tensor] = None
    o_b: Optional[torch.Tensor] = None


def _positions(ends: Sequence[int], lens: Sequence[int], device) -> torch.Tensor:
    """Where the last lens[b] tokens of sequences of ends[b] stand, packed."""
    parts = [torch.arange(end - n, end) for end, n in zip(ends, lens)]
    return (torch.cat(parts) if parts else torch.zeros(0, dtype=torch.int64)).to(device)


def _check_more(cache: str, had: Sequence[int], lens: Sequence[int]) -> None:
    if len(lens) != len(had):
        raise RuntimeError(f"{cache}: {len(lens)} sequences, the cache has {len(had)}")
    if any(n < 0 for n in lens):
        raise RuntimeError(f"{cache}: sequences grow by {list(lens)} tokens, none by fewer than 0")


class PackedCache:
    """Keys and values of several sequences, packed one after the other: per
    layer [sum(lens), kv_heads, dim]."""

    def __init__(self, layers: int, sequences: int):
        self.lens: List[int] = [0] * sequences
        self.k: List[Optional[torch.Tensor]] = [None] * layers
        self.v: List[Optional[torch.Tensor]] = [None] * layers
        self.old: Optional[torch.Tensor] = None
        self.new: Optional[torch.Tensor] = None
        self.cu: Optional[torch.Tensor] = None
        self.more: List[int] = [0] * sequences
        self.at: Optional[torch.Tensor] = None

    def grow(self, lens: Sequence[int], device) -> None:
        """Makes room for lens[b] tokens more of sequence b: where the kept and
        the new rows of each layer go."""
        _check_more("PackedCache", self.lens, lens)
        old, new, at, ends = [], [], 0, [0]
        for had, more in zip(self.lens, lens):
            old += range(at, at + had)
            new += range(at + had, at + had + more)
            at += had + more
            ends.append(at)
        self.old = torch.tensor(old, dtype=torch.int64, device=device)
        self.new = torch.tensor(new, dtype=torch.int64, device=device)
        self.cu = torch.tensor(ends, dtype=torch.int32, device=device)
        self.lens = [had + more for had, more in zip(self.lens, lens)]
        self.more, self.at = list(lens), None

    def positions(self, device) -> torch.Tensor:
        """Where the step's tokens stand in their sequences."""
        if self.at is None:
            self.at = _positions(self.lens, self.more, device)
        return self.at

    def state(self):
        """What restore() goes back to: grow() and add() put new tensors in their places and write none."""
        return list(self.lens), list(self.k), list(self.v), self.old, self.new, self.cu, self.more, self.at

    def restore(self, state) -> None:
        self.lens, self.k, self.v, self.old, self.new, self.cu, self.more, self.at = state

    def add(self, layer: int, k: torch.Tensor, v: torch.Tensor):
        if self.k[layer] is None:  # nothing kept: the new rows are the cache
            self.k[layer], self.v[layer] = k, v
        else:
            for store, rows in ((self.k, k), (self.v, v)):
                grown = rows.new_empty((sum(self.lens),) + rows.shape[1:])
                grown[self.old] = store[layer]
                grown[self.new] = rows
                store[layer] = grown
        return self.k[layer], self.v[layer]


class PagedCache:
    """Keys and values of several sequences in pages that every layer numbers
    alike: per layer [pages, page_size, kv_heads, dim].  Sequence b's token j is
    row j % page_size of page tables[b][j // page_size].  dtype: the rows' own
    type, or torch.float8_e4m3fn (a power of two beside each row)."""

    def __init__(self, layers: int, sequences: int, pages: int, kv_heads: int, dim: int, dtype: torch.dtype,
                 page_size: int = 64, device=None):
        if page_size < 16 or page_size & (page_size - 1):
            raise RuntimeError(f"PagedCache: page_size must be a power of two from 16 on, got {page_size}")
        shape = (pages, page_size, kv_heads, dim)
        # Rows that nothing wrote are never read as numbers; they need no clearing.
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.k_scales: List[Optional[torch.Tensor]] = [None] * layers
        self.v_scales: List[Optional[torch.Tensor]] = [None] * layers
        if dtype == torch.float8_e4m3fn:
            self.k_scales = [torch.empty(shape[:3], dtype=torch.uint8, device=device) for _ in range(layers)]
            self.v_scales = [torch.empty(shape[:3], dtype=torch.uint8, device=device) for _ in range(layers)]
        self.page_size = page_size
        self.lens: List[int] = [0] * sequences
        self.tables: List[List[int]] = [[] for _ in range(sequences)]
        self.free: List[int] = list(range(pages))
        self.slots: Optional[torch.Tensor] = None       # of the step's tokens
        self.positions: Optional[torch.Tensor] = None
        self.table: Optional[torch.Tensor] = None       # the step's, on the device
        self.kv_lens: Optional[torch.Tensor] = None

    def grow(self, lens: Sequence[int], device) -> None:
        """Takes the pages for lens[b] tokens more of sequence b."""
        _check_more("PagedCache", self.lens, lens)
        size = self.page_size
        ends = [had + more for had, more in zip(self.lens, lens)]
        need = [-(-end // size) - len(table) for end, table in zip(ends, self.tables)]
        if sum(need) > len(self.free):
            raise RuntimeError(f"PagedCache: the step takes {sum(need)} pages, {len(self.free)} are free")
        taken = iter(self.free[:sum(need)])
        self.free = self.free[sum(need):]
        self.tables = [table + [next(taken) for _ in range(n)] for table, n in zip(self.tables, need)]
        self.lens = ends
        rows = torch.zeros(len(ends), max([len(t) for t in self.tables], default=0), dtype=torch.int32)
        slots = []
        for b, (end, more) in enumerate(zip(ends, lens)):
            rows[b, :len(self.tables[b])] = torch.tensor(self.tables[b], dtype=torch.int32)
            at = torch.arange(end - more, end)
            slots.append(rows[b].long()[at // size] * size + at % size)
        self.slots = torch.cat(slots).to(device) if slots else torch.zeros(0, dtype=torch.int64, device=device)
        self.positions = _positions(ends, lens, device)
        self.table = rows.to(device)
        self.kv_lens = torch.tensor(ends, dtype=torch.int32, device=device)

    def cut(self, lens: Sequence[int]) -> None:
        """Keeps the first lens[b] tokens of sequence b (0: its place is free for
        another sequence); whole pages after them are free again."""
        if len(lens) != len(self.lens) or any(not 0 <= n <= had for n, had in zip(lens, self.lens)):
            raise RuntimeError(f"PagedCache: {list(lens)} tokens cannot stay of {self.lens}")
        keep = [-(-n // self.page_size) for n in lens]
        self.free = self.free + [page for table, n in zip(self.tables, keep) for page in table[n:]]
        self.tables = [table[:n] for table, n in zip(self.tables, keep)]
        self.lens = list(lens)

    def state(self):
        """What restore() goes back to: grow() puts new lists and tensors in their places and writes none."""
        return self.lens, self.tables, self.free, self.slots, self.positions, self.table, self.kv_lens

    def restore(self, state) -> None:
        self.lens, self.tables, self.free, self.slots, self.positions, self.table, self.kv_lens = state

    def layer(self, i: int):
        """(k_pages, v_pages) and the scales, as the engine's calls take them."""
        return (self.k[i], self.v[i]), dict(k_scales=self.k_scales[i], v_scales=self.v_scales[i])


Cache = Union[PackedCache, PagedCache]


class TenantDecoder:
    """layers: DecoderLayer weights in fp16 or bf16; embed [vocab, hidden];
    head [vocab, hidden].  Activations between layers keep the weights' type.
    rotary: how query and key heads turn with their positions (None: not).
    head_norms: per layer the weights [dim] of the query and the key heads' own
    norms, each a tensor or None."""

    def __init__(self, engine: WarpPipeEngine, embed: torch.Tensor, layers: Sequence[DecoderLayer], norm: torch.Tensor,
                 head: torch.Tensor, heads: int, kv_heads: int, scale: float = 1.0, eps: float = 1e-6,
                 rotary: Optional[Rotary] = None,
                 head_norms: Optional[Sequence[Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]]] = None):
        out = layers[0].w_qkv.size(0) if layers else 0
        if heads < 1 or kv_heads < 1 or heads % kv_heads != 0 or out % (heads + 2 * kv_heads) != 0:
            raise RuntimeError("TenantDecoder: w_qkv does not hold the query, key and value heads")
        if head_norms is not None and len(head_norms) != len(layers):
            raise RuntimeError(f"TenantDecoder: head_norms for {len(head_norms)} of {len(layers)} layers")
        self.head_norms = list(head_norms) if head_norms is not None else [(None, None)] * len(layers)
        self.engine, self.embed, self.layers, self.norm, self.head = engine, embed, list(layers), norm, head
        self.heads, self.kv_heads, self.dim = heads, kv_heads, out // (heads + 2 * kv_heads)
        self.scale, self.eps, self.rotary = float(scale), float(eps), rotary

    def paged_cache(self, sequences: int, pages: int, page_size: int = 64, dtype: Optional[torch.dtype] = None) -> PagedCache:
        """A cache for this model; dtype: the activations' unless given (torch.float8_e4m3fn: 8 bits)."""
        return PagedCache(len(self.layers), sequences, pages, self.kv_heads, self.dim,
                          self.embed.dtype if dtype is None else dtype, page_size, self.embed.device)

    def _rms(self, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        f = x.float()  # the mean square in fp32, one rounding at the end
        return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + self.eps) * weight.float()).to(x.dtype)

    def _lora(self, y, x, a, b) -> None:
        if a is not None and not self.engine.add_lora_packed(y, x, a, b, self.scale):
            raise RuntimeError(f"TenantDecoder: rank {a.size(2)} has no kernels")

    def _attend(self, i: int, qkv, cu_seqlens, cache: Cache):
        """The layer's attention; the heads are turned in qkv itself."""
        e, hq, hk = self.engine, self.heads, self.kv_heads
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        q_norm, k_norm = self.head_norms[i]
        turns = self.rotary is not None or q_norm is not None or k_norm is not None
        norms = dict(q_norm=q_norm, k_norm=k_norm, eps=self.eps)
        if isinstance(cache, PagedCache):
            pages, scales = cache.layer(i)
            if turns:
                e.rotate_into_cache(q, k, v, cache.positions, self.rotary, *pages, cache.slots, **scales, **norms, q_out=q)
            else:
                e.write_cache(k, v, *pages, cache.slots, **scales)
            return e.paged_attention(q, *pages, cache.table, cu_seqlens, cache.kv_lens, **scales)
        if turns:
            e.rotate_heads(q, k, cache.positions(q.device), self.rotary, **norms, q_out=q, k_out=k)
        k, v = cache.add(i, k, v)
        return e.packed_attention(q, k, v, cu_seqlens, cache.cu)

    def hidden(self, ids, cu_seqlens, tenants, cache: Cache) -> torch.Tensor:
        e, hq, hk, d = self.engine, self.heads, self.kv_heads, self.dim
        if not e.build_seg_bounds(tenants):
            raise RuntimeError(f"TenantDecoder: {ids.numel()} tokens exceed the engine's max_tokens")
        x = self.embed[ids]
        for i, w in enumerate(self.layers):
            n = self._rms(x, w.norm1)
            qkv = e.linear(n, w.w_qkv)
            self._lora(qkv, n, w.qkv_a, w.qkv_b)
            mix = self._attend(i, qkv.view(-1, hq + 2 * hk, d), cu_seqlens, cache).view(-1, hq * d)
            x = e.linear(mix, w.w_o, residual=x)
            self._lora(x, mix, w.o_a, w.o_b)
            n = self._rms(x, w.norm2)
            x = e.linear(e.linear(n, w.w_gate_up, activation="silu", gated=True), w.w_down, residual=x)
        return self._rms(x, self.norm)

    def score(self, ids, cu_seqlens, tenants, lens: Sequence[int], top: int = 0, cache: Optional[PagedCache] = None):
        """ids [tokens] int64: the prompts one after the other, lens[b] tokens
        each (cu_seqlens: their bounds on the device, int32); tenants [tokens]:
        each token's adapter (-1: none).  Returns (TokenLogprobs, cache): row t is
        about the token after token t, and names none at a prompt's end.  cache: a
        PagedCache to keep the prompts in, after what it holds (a new PackedCache
        unless given)."""
        if cache is None:
            cache = PackedCache(len(self.layers), len(lens))
        return self.verify(ids, cu_seqlens, tenants, lens, cache, top), cache

    def verify(self, ids, cu_seqlens, tenants, lens: Sequence[int], cache: Cache, top: int = 0) -> TokenLogprobs:
        """score() for tokens that follow what the cache holds; it keeps theirs
        too (a step that raises leaves it as it was)."""
        n = ids.numel()
        if sum(lens) != n or tenants.numel() != n or cu_seqlens.numel() != len(lens) + 1:
            raise RuntimeError(f"TenantDecoder: {n} tokens, {tenants.numel()} tenants, {cu_seqlens.numel()} bounds and "
                               f"lengths {list(lens)} do not go together")
        _check_more(type(cache).__name__, cache.lens, lens)
        # The token after each one: none at a sequence's end.  (An empty
        # sequence names its neighbour's last token, which ends too.)
        after = torch.roll(ids, -1)
        if n > 0:
            after[torch.tensor(lens).cumsum(0).sub(1).to(ids.device)] = -1
        kept = cache.state()
        try:
            cache.grow(lens, ids.device)
            hidden = self.hidden(ids, cu_seqlens, tenants, cache) if n > 0 else self.embed[:0]
            return self.engine.token_logprobs(self.engine.linear(hidden, self.head), after, top)
        except BaseException:
            cache.restore(kept)
            raise
