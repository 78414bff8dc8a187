"""Performance cases of the operators around the grouped LoRA apply: what a
program that serves or scores prompts under per-tenant adapters calls between
its LoRA deltas.

  linear            a projection with its bias, activation and residual
  packed_attention  attention over packed sequences of different lengths
  token_logprobs    what the model says of given tokens

A case is one call.  Its fields, by `op`:

  linear            tokens, d_in, d_out; act; gated: the weight holds d_out gate
                    rows and then d_out up rows, and the answer is
                    act(gate) * up; bias, residual: whether there is one
  packed_attention  kind "prompt": `batch` prompts of `tokens` tokens together,
                    q, k and v being views of one packed projection;
                    kind "cached": `batch` requests of `new` tokens (ragged: 0
                    to `new`) at the end of kv_min to kv_max cached keys;
                    heads, kv_heads, dim; window: keys that a query sees (0: all
                    up to its own); lengths: what the lengths are drawn from
  token_logprobs    tokens, vocab, top: alternatives per row; banned: the share
                    of the vocabulary that a mask has set to minus infinity

The plain forms compute in 32 bits and round once.
"""
import math
import random

import torch

own = False  # True: run() calls the framework's operators, else their plain forms

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    """The measured cases."""
    return [
        # The output projection of one decoding request, added to its residual
        # stream: the weight is read for a single row.
        dict(name="linear_token", op="linear", tokens=1, d_in=4096, d_out=4096, act="none", gated=False, bias=False,
             residual=True, dtype="bf16"),
        # A draft model's projection for 32 tenants of 4 tokens.
        dict(name="linear_draft", op="linear", tokens=128, d_in=2048, d_out=2048, act="silu", gated=False, bias=True,
             residual=False, dtype="bf16"),
        # A ragged prompt on a small model of odd widths.
        dict(name="linear_ragged", op="linear", tokens=777, d_in=1544, d_out=1101, act="gelu", gated=False, bias=True,
             residual=True, dtype="fp16"),
        # The gate and up projections of a decode batch.
        dict(name="linear_gated_512", op="linear", tokens=512, d_in=5120, d_out=13824, act="silu", gated=True,
             bias=False, residual=False, dtype="bf16"),
        # The same layer over a prefill chunk: the largest product of a step.
        dict(name="linear_gated_8192", op="linear", tokens=8192, d_in=5120, d_out=13824, act="silu", gated=True,
             bias=False, residual=False, dtype="bf16"),
        # One request's next token over a short cache: latency.
        dict(name="attention_token", op="packed_attention", kind="cached", batch=1, new=1, ragged=False, kv_min=777,
             kv_max=777, heads=32, kv_heads=8, dim=128, window=0, lengths=1, dtype="bf16"),
        # Verification of 4 drafted tokens for each of 32 tenants, some of whom
        # have fewer or none in this step; a small model of narrow heads.
        dict(name="attention_verify", op="packed_attention", kind="cached", batch=32, new=5, ragged=True, kv_min=33,
             kv_max=2500, heads=32, kv_heads=4, dim=64, window=0, lengths=2, dtype="fp16"),
        # A decode batch over caches from one key to 8192.
        dict(name="attention_decode", op="packed_attention", kind="cached", batch=64, new=1, ragged=False, kv_min=1,
             kv_max=8192, heads=32, kv_heads=8, dim=128, window=0, lengths=3, dtype="bf16"),
        # A prefill chunk of 16 prompts, every head with its own keys.
        dict(name="attention_prompts", op="packed_attention", kind="prompt", batch=16, tokens=8192, heads=32,
             kv_heads=32, dim=128, window=0, lengths=4, dtype="fp16"),
        # One long prompt.
        dict(name="attention_long", op="packed_attention", kind="prompt", batch=1, tokens=16384, heads=32, kv_heads=8,
             dim=128, window=0, lengths=5, dtype="bf16"),
        # Log probabilities of four requests' sampled tokens.
        dict(name="logprobs_token", op="token_logprobs", tokens=4, vocab=32000, top=5, banned=0.0, dtype="fp32"),
        # A prompt scored over a large vocabulary, with alternatives.
        dict(name="logprobs_prompt", op="token_logprobs", tokens=4096, vocab=128000, top=20, banned=0.01,
             dtype="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step`, uniform over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    """One more case of the listed ones' ranges."""
    most = {"linear": 0.0, "packed_attention": 0.0, "token_logprobs": 0.0}
    for c in listed():
        most[c["op"]] = max(most[c["op"]], _cost(c))
    while True:
        op = rng.choice(("linear", "packed_attention", "token_logprobs"))
        if op == "linear":
            case = dict(op=op, tokens=_log(rng, 1, 8192), d_in=_log(rng, 256, 8192, 1 if rng.random() < 0.15 else 8),
                        d_out=_log(rng, 256, 14336, rng.choice((1, 16))),
                        act=rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")), gated=rng.random() < 0.3,
                        bias=rng.random() < 0.5, residual=rng.random() < 0.5, dtype=rng.choice(("fp16", "bf16")))
        elif op == "packed_attention":
            kv = rng.choice((1, 2, 4, 8, 16))
            case = dict(op=op, kind=rng.choice(("prompt", "cached")), batch=_log(rng, 1, 64))
            if case["kind"] == "prompt":
                case["tokens"] = max(case["batch"], _log(rng, 16, 16384))
            else:
                case.update(new=_log(rng, 1, 512), ragged=rng.random() < 0.5, kv_min=_log(rng, 1, 512))
                case["kv_min"] = max(case["kv_min"], 1)
                case["kv_max"] = max(case["kv_min"], _log(rng, 64, 16384))
            case.update(heads=kv * rng.choice((1, 2, 3, 4, 7, 8)), kv_heads=kv, dim=rng.choice((64, 80, 96, 128, 128)),
                        window=rng.choice((0, 0, 0, _log(rng, 32, 4096))), lengths=rng.randrange(1 << 20),
                        dtype=rng.choice(("fp16", "bf16")))
        else:
            case = dict(op=op, tokens=_log(rng, 1, 4096), vocab=_log(rng, 1000, 200000),
                        top=rng.choice((0, 1, 5, 20, rng.randint(2, 32))), banned=rng.choice((0.0, 0.01, 0.9)),
                        dtype=rng.choice(("fp16", "bf16", "fp32")))
        if _cost(case) <= most[op]:
            return case


def _cost(case):
    """What the plain form of a case goes by: its products, scores or logits."""
    if case["op"] == "linear":
        return case["tokens"] * case["d_in"] * case["d_out"] * (2.0 if case["gated"] else 1.0)
    if case["op"] == "token_logprobs":
        return float(case["tokens"] * case["vocab"])
    lq, lk = _lengths(case)
    return float(len(lq) * max(lq) * max(lk) * case["heads"])


# ------------------------------------------------------------------ inputs --

def _lengths(case):
    """Each sequence's new tokens and keys."""
    r = random.Random(case["lengths"])
    n = case["batch"]
    if case["kind"] == "prompt":
        share = [math.exp(r.gauss(0.0, 1.0)) for _ in range(n)]
        lens = [1 + int(s / sum(share) * (case["tokens"] - n)) for s in share]
        lens[0] += case["tokens"] - sum(lens)
        return lens, lens
    lk = [_log(r, case["kv_min"], case["kv_max"]) for _ in range(n)]
    if n > 1:
        lk[0], lk[n // 2] = case["kv_max"], case["kv_min"]
    lq = [r.randint(0, case["new"]) if case["ragged"] else case["new"] for _ in range(n)]
    lq[0] = case["new"]
    # The new tokens' own keys are among the cached ones.
    return lq, [max(a, b) for a, b in zip(lq, lk)]


def _normal(shape, std, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFF)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def prepare(case, seed):
    seed = int(seed) * 16
    dt = _DT[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "linear":
        rows = case["d_out"] * (2 if case["gated"] else 1)
        s["x"] = _normal((case["tokens"], case["d_in"]), 1.0, dt, seed)
        s["weight"] = _normal((rows, case["d_in"]), 0.02, dt, seed + 1)
        s["bias"] = _normal((rows,), 0.5, dt, seed + 2) if case["bias"] else None
        s["residual"] = _normal((case["tokens"], case["d_out"]), 1.0, dt, seed + 3) if case["residual"] else None
    elif case["op"] == "packed_attention":
        lq, lk = _lengths(case)
        hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
        if case["kind"] == "prompt":
            qkv = _normal((sum(lq), hq + 2 * hk, d), 1.0, dt, seed)
            s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        else:
            s["q"] = _normal((sum(lq), hq, d), 1.0, dt, seed)
            s["k"] = _normal((sum(lk), hk, d), 1.0, dt, seed + 1)
            s["v"] = _normal((sum(lk), hk, d), 1.0, dt, seed + 2)
        s["lens_q"], s["lens_k"] = lq, lk
        ends = [torch.tensor(v).cumsum(0).to(torch.int32) for v in (lq, lk)]
        s["cu_q"], s["cu_k"] = (torch.cat([torch.zeros(1, dtype=torch.int32), e]).cuda() for e in ends)
    else:
        T, V = case["tokens"], case["vocab"]
        logits = _normal((T, V), 2.5, torch.float32, seed)
        g = torch.Generator(device="cuda").manual_seed((seed + 1) & 0x7FFFFFFF)
        ids = torch.randint(0, V, (T,), generator=g, device="cuda")
        if case["banned"]:
            off = torch.rand(V, generator=g, device="cuda") < case["banned"]
            logits[:, off] = -math.inf
        # Most given tokens are likely ones.
        likely = torch.rand(T, generator=g, device="cuda") < 0.8
        logits[torch.arange(T, device="cuda"), ids] = torch.where(likely, 12.0, 1.0) + 2.5 * torch.randn(
            T, generator=g, device="cuda")
        s["logits"], s["ids"] = logits.to(dt), ids
    return s


# ---------------------------------------------------------------- the calls --

_held = {}


def _engine():
    """The program's engine, made at its first call."""
    if "engine" not in _held:
        from adapterslotsplusplus_amd import WarpPipeEngine
        _held["engine"] = WarpPipeEngine()
    return _held["engine"]


def run(s):
    case = s["case"]
    if case["op"] == "linear":
        if own:
            return _engine().linear(s["x"], s["weight"], bias=s["bias"], residual=s["residual"], activation=case["act"],
                                    gated=case["gated"])
        return _plain_linear(s["x"], s["weight"], s["bias"], s["residual"], case["act"], case["gated"])
    if case["op"] == "packed_attention":
        if own:
            out, lse = _engine().packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], window=case["window"],
                                                  return_lse=True)
        else:
            out, lse = _plain_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max(s["lens_q"]),
                                        max(s["lens_k"]), case["window"])
        return {"out": out, "lse": lse}
    if own:
        got = _engine().token_logprobs(s["logits"], s["ids"], top=case["top"])
    else:
        got = _plain_logprobs(s["logits"], s["ids"], case["top"])
    return dict(zip(("logprobs", "entropy", "ranks", "top_logprobs", "top_ids"), got))


def _activate(a, act):
    if act == "relu":
        return a.clamp_min(0)
    if act == "gelu":
        return 0.5 * a * (1 + torch.erf(a * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a * a * a)))
    if act == "silu":
        return a / (1 + torch.exp(-a))
    return a


def _plain_linear(x, weight, bias, residual, act, gated):
    y = torch.matmul(x.float(), weight.float().t())
    if bias is not None:
        y = y + bias.float()
    if gated:
        n = y.size(1) // 2
        y = _activate(y[:, :n], act) * y[:, n:]
    else:
        y = _activate(y, act)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def _padded(t, cu, longest):
    """[B, longest, ...] of the packed t in 32 bits, and which places hold a token."""
    at = torch.arange(longest, device=t.device)
    held = at < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None].long() + at).clamp_max(max(t.size(0) - 1, 0))
    return t[rows].float(), held


def _plain_attention(q, k, v, cu_q, cu_k, longest_q, longest_k, window):
    B, (T, hq, d), hk = cu_q.numel() - 1, q.shape, k.size(1)
    group = hq // hk
    qp, q_held = _padded(q, cu_q, longest_q)
    kp, k_held = _padded(k, cu_k, longest_k)
    vp, _ = _padded(v, cu_k, longest_k)
    qp = qp.view(B, longest_q, hk, group, d).permute(0, 2, 3, 1, 4).reshape(B, hk, group * longest_q, d)
    scores = torch.matmul(qp, kp.permute(0, 2, 3, 1).contiguous()).mul_(1.0 / math.sqrt(d))
    # Position of each query among its sequence's keys: the last is at the end.
    after = ((cu_k[1:] - cu_k[:-1]) - (cu_q[1:] - cu_q[:-1]))[:, None] + torch.arange(longest_q, device=q.device)
    at = torch.arange(longest_k, device=q.device)
    seen = (at <= after[:, :, None]) & k_held[:, None, :]
    if window:
        seen &= at > after[:, :, None] - window
    scores = scores.view(B, hk, group, longest_q, longest_k)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, hk, group * longest_q, longest_k), vp.permute(0, 2, 1, 3).contiguous())
    out = out.view(B, hk, group, longest_q, d) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, longest_q, hq, d)
    lse = lse.permute(0, 3, 1, 2).reshape(B, longest_q, hq)
    return out[q_held].to(q.dtype), lse[q_held]


def _plain_logprobs(logits, ids, top):
    x = logits.float()
    most = x.amax(-1, keepdim=True)
    e = torch.exp(x - most)
    total = e.sum(-1, keepdim=True)
    lse = most + torch.log(total)
    given = x.gather(1, ids[:, None])
    logprobs = (given - lse).squeeze(1)
    weighted = torch.where(e > 0, e * (x - most), 0.0).sum(-1, keepdim=True)
    entropy = (torch.log(total) - weighted / total).squeeze(1)
    ranks = (x > given).sum(-1).add(1).to(torch.int32)
    # Values in order and, among equal ones, the lowest index first: one
    # whole number that holds both.
    bits = torch.where(x == 0, 0.0, x).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits + (1 << 31)))
    key = order * (1 << 32) + (x.size(1) - 1 - torch.arange(x.size(1), device=x.device))
    top_ids = (x.size(1) - 1 - key.topk(top, dim=1).values.remainder(1 << 32)).to(torch.int32)
    return logprobs, entropy, ranks, x.gather(1, top_ids.long()) - lse, top_ids


# --------------------------------------------------------------------- work --

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["d_in"], case["d_out"]
        rows = n * (2 if case["gated"] else 1)
        moved = t * k + rows * k + t * n * (2 if case["residual"] else 1) + (rows if case["bias"] else 0)
        return {"bytes": float(size * moved), "flops": 2.0 * t * k * rows}
    if case["op"] == "token_logprobs":
        t, v, top = case["tokens"], case["vocab"], case["top"]
        return {"bytes": float(t * (v * size + 8 + 12 + 8 * top)), "flops": 6.0 * t * v}
    lq, lk = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = keys = 0
    for a, b in zip(lq, lk):
        seen = b - a + 1  # the first query's keys
        w = case["window"] or b
        full = max(0, min(a, w - seen + 1))  # queries that see fewer keys than the window holds
        pairs += full * seen + full * (full - 1) // 2 + (a - full) * w
        keys += min(b, w + a - 1) if a else 0
    return {"bytes": float(size * d * (2 * sum(lq) * hq + 2 * keys * hk) + 4 * sum(lq) * hq),
            "flops": 4.0 * pairs * d * hq}


# -------------------------------------------------------------------- exact --

def exact(case, seed):
    """run()'s answer by the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s, case)
    if case["op"] == "packed_attention":
        return _exact_attention(s, case)
    return _exact_logprobs(s, case)


def _exact_linear(s, case):
    parts = []
    for x in s["x"].split(1024):
        y = x.double() @ s["weight"].double().t()
        if s["bias"] is not None:
            y += s["bias"].double()
        g = y[:, :case["d_out"]]
        if case["act"] == "relu":
            z = torch.relu(g)
        elif case["act"] == "gelu":
            z = g * torch.special.ndtr(g)
        elif case["act"] == "gelu_tanh":
            z = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        elif case["act"] == "silu":
            z = g * torch.sigmoid(g)
        else:
            z = g
        parts.append(z * y[:, case["d_out"]:] if case["gated"] else z)
    y = torch.cat(parts)
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_attention(s, case):
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    T = s["q"].size(0)
    out = torch.zeros(T, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device="cuda")
    at_q = at_k = 0
    for n_q, n_k in zip(s["lens_q"], s["lens_k"]):
        for first in range(0, n_q, 1024):
            rows = torch.arange(first, min(n_q, first + 1024), device="cuda")
            pos = rows + n_k - n_q
            lo = max(0, int(first + n_k - n_q) - case["window"] + 1) if case["window"] else 0
            hi = min(n_k, first + len(rows) + n_k - n_q)
            keys = torch.arange(lo, hi, device="cuda")
            hide = keys[None] > pos[:, None]
            if case["window"]:
                hide |= keys[None] <= pos[:, None] - case["window"]
            for h in range(hk):
                kk = s["k"][at_k + lo:at_k + hi, h].double()
                vv = s["v"][at_k + lo:at_k + hi, h].double()
                for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                    z = s["q"][at_q + rows, g].double() @ kk.t().contiguous() / math.sqrt(d)
                    z = z.masked_fill(hide, -math.inf)
                    out[at_q + rows, g] = torch.softmax(z, -1) @ vv
                    lse[at_q + rows, g] = torch.logsumexp(z, -1)
        at_q, at_k = at_q + n_q, at_k + n_k
    return {"out": out, "lse": lse}


def _exact_logprobs(s, case):
    V, top = case["vocab"], case["top"]
    got = []
    for x, ids in zip(s["logits"].split(256), s["ids"].split(256)):
        logp = torch.log_softmax(x.double(), -1)
        given = logp.gather(1, ids[:, None])
        entropy = -(logp.exp() * logp.masked_fill(logp == -math.inf, 0.0)).sum(-1)
        ranks = 1 + (x > x.gather(1, ids[:, None])).sum(-1)
        at = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
        got.append((given.squeeze(1), entropy, ranks.to(torch.int32), logp.gather(1, at), at.to(torch.int32)))
    assert V == s["logits"].size(1)
    return dict(zip(("logprobs", "entropy", "ranks", "top_logprobs", "top_ids"), (torch.cat(p) for p in zip(*got))))
