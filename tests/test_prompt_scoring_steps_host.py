"""Host-side: a decoder's steps on an engine that computes on the CPU (no GPU):
what a step that fails leaves of the cache."""
import pytest
import torch

from adapterslotsplusplus_amd.engine import TokenLogprobs
from adapterslotsplusplus_amd.prompt_scoring import DecoderLayer, TenantDecoder

HEADS, KV, DIM, VOCAB = 2, 1, 8, 11


class HostEngine:
    """Plain operators; `refuse` names the call that answers as the engine does when it cannot."""

    def __init__(self, refuse=None):
        self.refuse, self.calls = refuse, 0

    def build_seg_bounds(self, tenants):
        return self.refuse != "tokens"

    def add_lora_packed(self, y, x, a, b, scale):
        self.calls += 1
        return not (self.refuse == "rank" and self.calls > 1)  # the second projection's

    def linear(self, x, w, bias=None, residual=None, activation="none", gated=False):
        y = x @ w.t()
        if gated:
            y = torch.nn.functional.silu(y[:, :y.size(1) // 2]) * y[:, y.size(1) // 2:]
        return y if residual is None else y + residual

    def packed_attention(self, q, k, v, cu_q, cu_k):
        out = torch.zeros(q.shape)
        for b in range(len(cu_q) - 1):
            qq, kk, vv = q[cu_q[b]:cu_q[b + 1]], k[cu_k[b]:cu_k[b + 1]], v[cu_k[b]:cu_k[b + 1]]
            n, m = len(qq), len(kk)
            hide = torch.arange(m) > torch.arange(n)[:, None] + m - n
            for h in range(HEADS):
                s = (qq[:, h] @ kk[:, 0].t()) * DIM ** -0.5
                out[cu_q[b]:cu_q[b + 1], h] = torch.softmax(s.masked_fill(hide, float("-inf")), -1) @ vv[:, 0]
        return out

    def token_logprobs(self, logits, ids, top=0):
        if self.refuse == "top":
            raise RuntimeError("token_logprobs: refused")
        lp = torch.log_softmax(logits, -1)
        given = torch.where(ids >= 0, lp.gather(1, ids.clamp(min=0)[:, None])[:, 0], 0.0)
        return TokenLogprobs(given, given, given, given.new_zeros(len(ids), top), given.new_zeros(len(ids), top))


def decoder(engine, layers=2):
    g = torch.Generator().manual_seed(0)

    def w(*shape):
        return torch.randn(*shape, generator=g) * 0.3

    ls = [DecoderLayer(w(16), w((HEADS + 2 * KV) * DIM, 16), w(16, HEADS * DIM), w(16), w(40, 16), w(16, 20),
                       w(1, 1, 8, 16), w(1, 1, 32, 8), w(1, 1, 8, 16), w(1, 1, 16, 8)) for _ in range(layers)]
    return TenantDecoder(engine, w(VOCAB, 16), ls, w(16), w(VOCAB, 16), HEADS, KV)


def step(model, parts, cache=None):
    lens = [len(p) for p in parts]
    ids = torch.cat(parts)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    who = torch.zeros(len(ids), dtype=torch.int64)
    return model.score(ids, cu, who, lens) if cache is None else model.verify(ids, cu, who, lens, cache)


def parts(seed, *lens):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (n,), generator=g) for n in lens]


@pytest.mark.parametrize("refuse,message", [("tokens", "max_tokens"), ("rank", "no kernels"), ("top", "refused")])
def test_a_step_that_fails_leaves_the_cache(refuse, message):
    engine = HostEngine()
    model = decoder(engine)
    first, more = parts(1, 3, 0, 5), parts(2, 2, 4, 1)
    _, cache = step(model, first)
    want = step(decoder(HostEngine()), more, step(decoder(HostEngine()), first)[1])
    engine.refuse, engine.calls = refuse, 0
    with pytest.raises(RuntimeError, match=message):
        step(model, more, cache)
    assert cache.lens == [3, 0, 5] and all(len(t) == 8 for t in cache.k + cache.v)
    engine.refuse = None
    got = step(model, more, cache)
    assert torch.equal(got.logprobs, want.logprobs) and cache.lens == [5, 4, 6]


def test_a_batch_of_another_size_leaves_the_cache():
    model = decoder(HostEngine())
    _, cache = step(model, parts(1, 3, 2))
    with pytest.raises(RuntimeError, match="1 sequences"):
        step(model, parts(2, 1), cache)
    assert cache.lens == [3, 2] and all(len(t) == 5 for t in cache.k + cache.v)


def test_steps_of_no_tokens():
    """On a new cache and between steps that have some; they change nothing."""
    model = decoder(HostEngine())
    got, cache = step(model, parts(0, 0, 0))
    assert got.logprobs.shape == (0,) and cache.lens == [0, 0]
    first, more = parts(1, 0, 4), parts(2, 2, 3)
    step(model, first, cache)
    assert step(model, parts(0, 0, 0), cache).logprobs.shape == (0,)
    got = step(model, more, cache)
    want = step(model, more, step(model, first)[1])
    assert torch.equal(got.logprobs, want.logprobs) and cache.lens == [2, 7]


def test_lengths_must_cover_the_tokens():
    model = decoder(HostEngine())
    ids, cu, who = torch.arange(5), torch.tensor([0, 2, 5], dtype=torch.int32), torch.zeros(5, dtype=torch.int64)
    for bad in ((ids, cu, who, [2, 4]), (ids, cu, who, [5]), (ids, cu, who[:4], [2, 3]), (ids[:4], cu, who[:4], [2, 3])):
        with pytest.raises(RuntimeError, match="do not go together"):
            model.score(*bad)
