"""A multi-tenant decoder on the engine's operators: what a model says of
given tokens, every token under its own tenant's adapters.

`TenantDecoder` is a stack of pre-norm decoder layers whose projections run on
`engine.linear` (the gated MLP's two projections and their product in one
launch, residuals added in the epilogue), whose attention runs on
`engine.packed_attention` over the packed prompts, and whose logits are read
once by `engine.token_logprobs`.  The adapters' deltas are
`engine.add_lora_packed` calls on the step's one segment table.

  * `score(ids, cu_seqlens, tenants)`: per token the log probability of the one
    after it -- scoring prompts, or the first step of a request (it leaves the
    prompts' keys and values in a `PackedCache`);
  * `verify(ids, cu_seqlens, tenants, cache)`: the same for tokens drafted after
    what the cache holds, all in one pass; the cache grows by them.

Nothing here waits for the device; the lengths that the caller passes, and
where the cache's rows go, are uploaded from host memory at each step.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence

import torch

from .engine import TokenLogprobs, WarpPipeEngine


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

    def grow(self, lens: Sequence[int], device) -> None:
        """Makes room for lens[b] tokens more of sequence b: where the kept and
        the new rows of each layer go."""
        if len(lens) != len(self.lens):
            raise RuntimeError(f"PackedCache: {len(lens)} sequences, the cache has {len(self.lens)}")
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

    def state(self):
        """What restore() goes back to: grow() and add() put new tensors in their places and write none."""
        return list(self.lens), list(self.k), list(self.v), self.old, self.new, self.cu

    def restore(self, state) -> None:
        self.lens, self.k, self.v, self.old, self.new, self.cu = state

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


class TenantDecoder:
    """layers: DecoderLayer weights in fp16 or bf16; embed [vocab, hidden];
    head [vocab, hidden].  Activations between layers keep the weights' type."""

    def __init__(self, engine: WarpPipeEngine, embed: torch.Tensor, layers: Sequence[DecoderLayer], norm: torch.Tensor,
                 head: torch.Tensor, heads: int, kv_heads: int, scale: float = 1.0, eps: float = 1e-6):
        out = layers[0].w_qkv.size(0) if layers else 0
        if heads < 1 or kv_heads < 1 or heads % kv_heads != 0 or out % (heads + 2 * kv_heads) != 0:
            raise RuntimeError("TenantDecoder: w_qkv does not hold the query, key and value heads")
        self.engine, self.embed, self.layers, self.norm, self.head = engine, embed, list(layers), norm, head
        self.heads, self.kv_heads, self.dim = heads, kv_heads, out // (heads + 2 * kv_heads)
        self.scale, self.eps = float(scale), float(eps)

    def _rms(self, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        f = x.float()  # the mean square in fp32, one rounding at the end
        return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + self.eps) * weight.float()).to(x.dtype)

    def _lora(self, y, x, a, b) -> None:
        if a is not None and not self.engine.add_lora_packed(y, x, a, b, self.scale):
            raise RuntimeError(f"TenantDecoder: rank {a.size(2)} has no kernels")

    def hidden(self, ids, cu_seqlens, tenants, cache: PackedCache) -> torch.Tensor:
        e, hq, hk, d = self.engine, self.heads, self.kv_heads, self.dim
        if not e.build_seg_bounds(tenants):
            raise RuntimeError(f"TenantDecoder: {ids.numel()} tokens exceed the engine's max_tokens")
        x = self.embed[ids]
        for i, w in enumerate(self.layers):
            n = self._rms(x, w.norm1)
            qkv = e.linear(n, w.w_qkv)
            self._lora(qkv, n, w.qkv_a, w.qkv_b)
            qkv = qkv.view(-1, hq + 2 * hk, d)
            k, v = cache.add(i, qkv[:, hq:hq + hk], qkv[:, hq + hk:])
            mix = e.packed_attention(qkv[:, :hq], k, v, cu_seqlens, cache.cu).view(-1, hq * d)
            x = e.linear(mix, w.w_o, residual=x)
            self._lora(x, mix, w.o_a, w.o_b)
            n = self._rms(x, w.norm2)
            x = e.linear(e.linear(n, w.w_gate_up, activation="silu", gated=True), w.w_down, residual=x)
        return self._rms(x, self.norm)

    def score(self, ids, cu_seqlens, tenants, lens: Sequence[int], top: int = 0):
        """ids [tokens] int64: the prompts one after the other, lens[b] tokens
        each (cu_seqlens: their bounds on the device, int32); tenants [tokens]:
        each token's adapter (-1: none).  Returns (TokenLogprobs, PackedCache):
        row t is about the token after token t, and names none at a prompt's end."""
        cache = PackedCache(len(self.layers), len(lens))
        return self.verify(ids, cu_seqlens, tenants, lens, cache, top), cache

    def verify(self, ids, cu_seqlens, tenants, lens: Sequence[int], cache: PackedCache, top: int = 0) -> TokenLogprobs:
        """score() for tokens that follow what the cache holds; it keeps theirs
        too (a step that raises leaves it as it was)."""
        n = ids.numel()
        if sum(lens) != n or tenants.numel() != n or cu_seqlens.numel() != len(lens) + 1:
            raise RuntimeError(f"TenantDecoder: {n} tokens, {tenants.numel()} tenants, {cu_seqlens.numel()} bounds and "
                               f"lengths {list(lens)} do not go together")
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
