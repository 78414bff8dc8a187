"""GPU: the multi-tenant decoder against the same model in plain 64-bit math.

Tolerance: the plain model is evaluated twice, once with every activation
rounded to the tensors' type where the operators round and once with none.
How far the two differ is what those roundings do to this model; a pass that
rounds at the same places, its sums in another order, may differ from the
unrounded one by as much again and the same once more for its own rounding
pattern (each is one draw of the same errors): three times their largest difference.
"""
import math

import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from adapterslotsplusplus_amd.prompt_scoring import DecoderLayer, TenantDecoder
from oracle import model_ops as mo
from tests.helpers import announce, gen

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, FFN, VOCAB, RANK, TENANTS, EPS = 256, 4, 2, 64, 512, 1003, 16, 3, 1e-6


def weights(dtype, layers, seed):
    g = gen(seed)

    def w(*shape, std):
        return (torch.randn(*shape, generator=g) * std).to(dtype)

    qkv = (HEADS + 2 * KV) * DIM
    ls = [DecoderLayer(1 + w(HIDDEN, std=0.1), w(qkv, HIDDEN, std=HIDDEN ** -0.5), w(HIDDEN, HEADS * DIM, std=0.05),
                       1 + w(HIDDEN, std=0.1), w(2 * FFN, HIDDEN, std=HIDDEN ** -0.5), w(HIDDEN, FFN, std=0.05),
                       w(TENANTS, 1, RANK, HIDDEN, std=HIDDEN ** -0.5), w(TENANTS, 1, qkv, RANK, std=0.1),
                       w(TENANTS, 1, RANK, HEADS * DIM, std=0.06), w(TENANTS, 1, HIDDEN, RANK, std=0.1))
          for _ in range(layers)]
    return w(VOCAB, HIDDEN, std=1.0), ls, 1 + w(HIDDEN, std=0.1), w(VOCAB, HIDDEN, std=0.1)


def plain(embed, layers, norm, head, ids, tenants, lens, dtype):
    """The model in 64 bits; dtype: activations rounded to it, None: not."""
    def r(t):
        return t if dtype is None else t.to(dtype).double()

    def rms(x, w):
        return r(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double())

    def lora(y, x, a, b):
        d = torch.zeros_like(y)
        for t, i in enumerate(tenants):
            if i >= 0:
                d[t] = b[i, 0].double() @ (a[i, 0].double() @ x[t])
        return r(y + d)

    x = embed.double()[ids]
    for w in layers:
        n = rms(x, w.norm1)
        qkv = lora(r(n @ w.w_qkv.double().T), n, w.qkv_a, w.qkv_b).view(len(ids), -1, DIM)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:]
        mix = r(mo.attention(q, k, v, lens, lens, DIM ** -0.5)[0].reshape(len(ids), -1))
        x = lora(r(mix @ w.w_o.double().T + x), mix, w.o_a, w.o_b)
        n = rms(x, w.norm2)
        gate, up = (n @ w.w_gate_up.double().T).chunk(2, -1)
        x = r(r(mo.activate(gate, "silu") * up) @ w.w_down.double().T + x)
    return torch.log_softmax(r(rms(x, norm) @ head.double().T), -1)


def on_gpu(m):
    embed, layers, norm, head = m
    return embed.cuda(), [DecoderLayer(*(t.cuda() for t in w)) for w in layers], norm.cuda(), head.cuda()


def bounds(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_prompts_and_drafts(dtype):
    announce(f"prompt scoring {dtype}")
    m = weights(dtype, 2, 11)
    prompts, drafts = [37, 1, 90, 5], [3, 4, 1, 2]
    g = gen(5)
    ids = [torch.randint(0, VOCAB, (a + b,), generator=g) for a, b in zip(prompts, drafts)]
    whole = [len(s) for s in ids]
    who = [0, 1, -1, 2]
    flat, tenants = torch.cat(ids), [t for t, n in zip(who, whole) for _ in range(n)]
    exact = plain(*m, flat, tenants, whole, None)
    slack = 3 * (plain(*m, flat, tenants, whole, dtype) - exact).abs().max().item()
    assert 0 < slack < 0.5

    embed, layers, norm, head = on_gpu(m)
    model = TenantDecoder(WarpPipeEngine(), embed, layers, norm, head, HEADS, KV, eps=EPS)

    def run(parts, lens, cache=None):
        x = torch.cat(parts).cuda()
        t = torch.tensor([t for t, n in zip(who, lens) for _ in range(n)]).cuda()
        if cache is None:
            return model.score(x, bounds(lens), t, lens, top=5)
        return model.verify(x, bounds(lens), t, lens, cache, top=5), cache

    def check(got, rows, parts):
        after = torch.cat([torch.cat([p[1:], torch.tensor([-1])]) for p in parts])
        want = torch.where(after >= 0, exact[rows].gather(1, after.clamp(min=0)[:, None])[:, 0], 0.0)
        assert ((got.logprobs.double().cpu() - want).abs() <= slack).all()
        assert ((got.top_logprobs.double().cpu() - exact[rows].gather(1, got.top_ids.long().cpu())).abs() <= slack).all()
        best = exact[rows].topk(5).values
        assert ((got.top_logprobs.double().cpu() - best).abs() <= slack).all()
        entropy = -(exact[rows].exp() * exact[rows]).sum(-1)
        # dH = -sum dp (log p + H): at most the slack times the mean of |log p + H|, and that once more for p's own change.
        reach = (exact[rows].exp() * (exact[rows] + entropy[:, None]).abs()).sum(-1)
        assert ((got.entropy.double().cpu() - entropy).abs() <= slack * (1 + reach) * math.exp(slack)).all()

    starts = [sum(whole[:b]) for b in range(len(whole))]
    got, _ = run(ids, whole)
    check(got, torch.arange(len(flat)), ids)
    first = [s[:n] for s, n in zip(ids, prompts)]
    rest = [s[n:] for s, n in zip(ids, prompts)]
    got, cache = run(first, prompts)
    check(got, torch.cat([torch.arange(n) + s for s, n in zip(starts, prompts)]), first)
    got, cache = run(rest, drafts, cache)
    check(got, torch.cat([torch.arange(d) + s + n for s, n, d in zip(starts, prompts, drafts)]), rest)
    assert cache.lens == whole
