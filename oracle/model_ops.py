"""The operators around the LoRA apply by their definitions, in 64 bits on the
CPU: a projection with its epilogue, attention over packed sequences, and what
logits say of given tokens."""
from __future__ import annotations

import math

import torch


def activate(a: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.where(a < 0, torch.zeros_like(a), a)
    if act == "gelu":
        return 0.5 * a * (1 + torch.erf(a / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
    if act == "silu":
        return a / (1 + torch.exp(-a))
    return a


def linear(x, weight, bias=None, residual=None, act="none", gated=False):
    """(y, size): y in 64 bits, and per element the sum of the magnitudes that
    its fp32 accumulation sees, which scales the error it may have."""
    x, w = x.double(), weight.double()
    a, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        a, s = a + bias.double(), s + bias.double().abs()
    if gated:
        n = a.size(1) // 2
        g, u = activate(a[:, :n], act), a[:, n:]
        a, s = g * u, s[:, :n] * u.abs() + g.abs() * s[:, n:]
    else:
        a = activate(a, act)
    if residual is not None:
        a, s = a + residual.double(), s + residual.double().abs()
    return a, s


def attention(q, k, v, lens_q, lens_k, scale, causal=True, window=0):
    """(out, lse, spread, reach): spread is sum p |v| / sum p, and reach the
    largest sum of |q| |k| * scale over a query's keys: what the errors of an
    fp32 evaluation scale with."""
    T, heads, dim = q.shape
    group = heads // k.size(1)
    out = torch.zeros(T, heads, dim, dtype=torch.float64)
    spread = torch.zeros(T, heads, dim, dtype=torch.float64)
    lse = torch.full((T, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros(T, heads, dtype=torch.float64)
    a = b = 0
    for n_q, n_k in zip(lens_q, lens_k):
        for i in range(n_q):
            pos = i + n_k - n_q
            end = max(0, min(n_k, pos + 1)) if causal else n_k
            first = max(0, pos - window + 1) if causal and window else 0
            if end <= first:
                continue
            kk, vv = (t[b + first:b + end].double().repeat_interleave(group, 1) for t in (k, v))
            qq = q[a + i].double()
            s = torch.einsum("hd,jhd->hj", qq, kk) * scale
            reach[a + i] = (torch.einsum("hd,jhd->hj", qq.abs(), kk.abs()) * abs(scale)).amax(1)
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - m)
            l = p.sum(1, keepdim=True)
            out[a + i] = torch.einsum("hj,jhd->hd", p, vv) / l
            spread[a + i] = torch.einsum("hj,jhd->hd", p, vv.abs()) / l
            lse[a + i] = (m + torch.log(l)).squeeze(1)
        a, b = a + n_q, b + n_k
    return out, lse, spread, reach


def token_logprobs(logits, ids, top):
    """(logprobs, entropy, ranks, top_logprobs, top_ids); logits hold no NaN."""
    x = logits.double()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    named = (ids >= 0) & (ids < x.size(1))
    given = x.gather(1, torch.where(named, ids, 0)[:, None].long())
    zero = torch.zeros((), dtype=torch.float64)
    logprobs = torch.where(named, (given - lse).squeeze(1), zero)
    ranks = torch.where(named, 1 + (x > given).sum(1), 0).to(torch.int32)
    entropy = (torch.log(total) - torch.where(e > 0, e * (x - m), zero).sum(1, keepdim=True) / total).squeeze(1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return logprobs, entropy, ranks, x.gather(1, order) - lse, order.to(torch.int32)
