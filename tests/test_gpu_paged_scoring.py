"""GPU: the multi-tenant decoder with normed and turned heads over a paged
cache, against the same model in plain 64-bit math.

Tolerance: the plain model is evaluated twice, once with every activation and
kept row rounded where the operators round and once with none.  How far the two
differ is what those roundings do to this model; a pass that rounds at the same
places, its sums in another order, may differ from the unrounded one by as much
again and the same once more for its own rounding pattern: three times their
largest difference.
"""
import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from adapterslotsplusplus_amd.prompt_scoring import TenantDecoder
from adapterslotsplusplus_amd.rotary import Rotary, frequencies
from oracle import cache_ops as co
from oracle import model_ops as mo
from tests.helpers import announce, gen
from tests.test_gpu_prompt_scoring import DIM, EPS, HEADS, KV, VOCAB, bounds, on_gpu, weights

pytestmark = pytest.mark.gpu

WHO = [0, 1, -1, 2]


def model_of(dtype):
    embed, layers, norm, head = weights(dtype, 2, 11)
    g = gen(12)
    norms = [tuple((1 + 0.1 * torch.randn(DIM, generator=g)).to(dtype) for _ in "qk") for _ in layers]
    return embed, layers, norm, head, norms


def plain(embed, layers, norm, head, norms, ids, tenants, lens, dtype, small):
    """The model in 64 bits; dtype: activations rounded to it, None: not.  small:
    keys and values as e4m3 rows hold them (keys not rounded to dtype before)."""
    def r(t):
        return t if dtype is None else t.to(dtype).double()

    def kept(t):
        return t if dtype is None else co.quantise(t, torch.finfo(dtype).max)[0] if small else r(t)

    def rms(x, w):
        return r(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double())

    def lora(y, x, a, b):
        d = torch.zeros_like(y)
        for t, i in enumerate(tenants):
            if i >= 0:
                d[t] = b[i, 0].double() @ (a[i, 0].double() @ x[t])
        return r(y + d)

    at = torch.cat([torch.arange(n) for n in lens])
    freq = frequencies(DIM)[0]
    x = embed.double()[ids]
    for w, (q_norm, k_norm) in zip(layers, norms):
        n = rms(x, w.norm1)
        qkv = lora(r(n @ w.w_qkv.double().T), n, w.qkv_a, w.qkv_b).view(len(ids), -1, DIM)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:]
        q = r(co.rotate(co.norm_heads(q, q_norm, EPS), at, freq))
        k, v = kept(co.rotate(co.norm_heads(k, k_norm, EPS), at, freq)), kept(v)
        mix = r(mo.attention(q, k, v, lens, lens, DIM ** -0.5)[0].reshape(len(ids), -1))
        x = lora(r(mix @ w.w_o.double().T + x), mix, w.o_a, w.o_b)
        n = rms(x, w.norm2)
        gate, up = (n @ w.w_gate_up.double().T).chunk(2, -1)
        x = r(r(mo.activate(gate, "silu") * up) @ w.w_down.double().T + x)
    return torch.log_softmax(r(rms(x, norm) @ head.double().T), -1)


def run(model, parts, cache):
    lens = [len(p) for p in parts]
    t = torch.tensor([t for t, n in zip(WHO, lens) for _ in range(n)]).cuda()
    return model.verify(torch.cat(parts).cuda(), bounds(lens), t, lens, cache, top=5)


def check(got, exact, parts, slack):
    """exact: the plain model's rows of the parts' tokens."""
    after = torch.cat([torch.cat([p[1:], torch.tensor([-1])]) if len(p) else p for p in parts])
    want = torch.where(after >= 0, exact.gather(1, after.clamp(min=0)[:, None])[:, 0], 0.0)
    assert ((got.logprobs.double().cpu() - want).abs() <= slack).all()
    assert ((got.top_logprobs.double().cpu() - exact.gather(1, got.top_ids.long().cpu())).abs() <= slack).all()
    assert ((got.top_logprobs.double().cpu() - exact.topk(5).values).abs() <= slack).all()


@pytest.mark.parametrize("kind", ["packed", "pages", "8bit"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_prompts_drafts_and_single_tokens(dtype, kind):
    announce(f"scoring over {kind} {dtype}")
    m = model_of(dtype)
    steps = [[37, 1, 90, 0], [3, 4, 0, 70], [1, 1, 1, 1]]
    whole = [sum(s) for s in zip(*steps)]
    g = gen(5)
    ids = [torch.randint(0, VOCAB, (n,), generator=g) for n in whole]
    flat, tenants = torch.cat(ids), [t for t, n in zip(WHO, whole) for _ in range(n)]
    exact = plain(*m, flat, tenants, whole, None, False)
    slack = 3 * (plain(*m, flat, tenants, whole, dtype, kind == "8bit") - exact).abs().max().item()
    assert 0 < slack < 3
    rows = exact.split(whole)

    embed, layers, norm, head = on_gpu(m[:4])
    engine = WarpPipeEngine()
    model = TenantDecoder(engine, embed, layers, norm, head, HEADS, KV, eps=EPS, rotary=Rotary(DIM),
                          head_norms=[tuple(t.cuda() for t in pair) for pair in m[4]])
    cache = None
    if kind != "packed":
        cache = model.paged_cache(4, pages=24, page_size=16, dtype=torch.float8_e4m3fn if kind == "8bit" else None)
        for t in cache.k + cache.v:  # what was never written is not read as numbers
            t.view(torch.uint8).fill_(0xff)
        cache.free = cache.free[::-1]
    had = [0] * 4
    for lens in steps:
        parts = [s[a:a + n] for s, a, n in zip(ids, had, lens)]
        if cache is None:
            t = torch.tensor([t for t, n in zip(WHO, lens) for _ in range(n)]).cuda()
            got, cache = model.score(torch.cat(parts).cuda(), bounds(lens), t, lens, top=5)
        else:
            got = run(model, parts, cache)
        check(got, torch.cat([r[a:a + n] for r, a, n in zip(rows, had, lens)]), parts, slack)
        had = [a + n for a, n in zip(had, lens)]
        assert cache.lens == had
    assert engine.device_errors() == 0

    if kind == "packed":
        return
    # Drafts that were taken back leave no trace, and a finished sequence's pages serve a new one.
    cache.cut([a - 2 if a > 40 else a for a in had])
    back = [s[a:] for s, a in zip(ids, cache.lens)]
    check(run(model, back, cache), torch.cat([r[len(r) - len(p):] for r, p in zip(rows, back)]), back, slack)
    cache.cut([had[0], had[1], 0, had[3]])
    back = [p[:0] if b != 2 else ids[2] for b, p in enumerate(ids)]
    check(run(model, back, cache), rows[2], back, slack)
    assert engine.device_errors() == 0
