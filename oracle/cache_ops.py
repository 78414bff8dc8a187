"""Rows of heads and a paged cache by their definitions, in 64 bits on the CPU:
norms and rotation by position, e4m3 rows with a power of two each, and
attention over pages."""
from __future__ import annotations

import math

import torch

from .model_ops import attention as _attention


def norm_heads(x, weight, eps):
    x = x.double()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()


def rotate(x, positions, frequencies, factor=1.0, interleaved=False):
    """x [tokens, heads, dim] in 64 bits, its first 2 * len(frequencies) elements
    turned by positions * frequencies radians."""
    x = x.double()
    f = torch.tensor(frequencies, dtype=torch.float64)
    h = f.numel()
    angle = positions.double()[:, None] * f
    c, s = (torch.cos(angle) * factor)[:, None], (torch.sin(angle) * factor)[:, None]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    u, w = a * c - b * s, b * c + a * s
    y = x.clone()
    if interleaved:
        y[..., 0:2 * h:2], y[..., 1:2 * h:2] = u, w
    else:
        y[..., :h], y[..., h:2 * h] = u, w
    return y


def e4m3(y):
    """y in 64 bits, rounded to the nearest value of 4 significant bits with
    exponents from -6 on, ties to even (|y| at most 464)."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(y / step) * step


def quantise(rows, largest):
    """(values, scale exponents) of rows [..., dim] whose type's largest finite
    value is `largest`: what a cache of e4m3 rows holds of them.  Finite
    magnitudes past that one count as it."""
    x = rows.double()
    finite = x.isfinite()
    x = torch.where(finite, x.clamp(-largest, largest), x)
    top = torch.where(finite, x.abs(), 0.0).amax(-1)
    e = torch.full(top.shape, -126, dtype=torch.int64)
    some = top > 0
    e[some] = torch.tensor([max(-126, math.frexp(t)[1] - 9 + (1 if math.frexp(t)[0] > 0.875 else 0)) for t in top[some].tolist()],
                           dtype=torch.int64)
    s = torch.exp2(e.double())[..., None]
    v = e4m3(torch.where(finite, x, 0.0) / s) * s
    # What would come back as an infinity takes the value of 4 bits below it.
    v = torch.where(v.abs() > largest, torch.sign(v) * 240 * s, v)
    return torch.where(finite, v, torch.nan), e


def paged_attention(q, k_pages, v_pages, block_table, lens_q, lens_k, scale, window=0, sinks=0):
    """model_ops.attention's (out, lse, spread, reach) over a cache of values
    [pages, page_size, kv_heads, dim] in 64 bits.  With a window, a query sees
    the first `sinks` keys too."""
    page = k_pages.size(1)
    rows = [torch.tensor([int(block_table[b, j // page]) * page + j % page for j in range(n)], dtype=torch.int64)
            for b, n in enumerate(lens_k)]
    k, v = (t.reshape(-1, *t.shape[2:])[torch.cat(rows) if rows else torch.zeros(0, dtype=torch.int64)] for t in (k_pages, v_pages))
    if not window or not sinks:
        return _attention(q, k, v, lens_q, lens_k, scale, True, window)
    T, heads, dim = q.shape
    group = heads // k.size(1)
    out, spread = torch.zeros(T, heads, dim, dtype=torch.float64), torch.zeros(T, heads, dim, dtype=torch.float64)
    lse, reach = torch.full((T, heads), -math.inf, dtype=torch.float64), torch.zeros(T, heads, dtype=torch.float64)
    a = b = 0
    for n_q, n_k in zip(lens_q, lens_k):
        for i in range(n_q):
            pos = i + n_k - n_q
            if pos < 0:
                continue
            at = torch.tensor([j for j in range(pos + 1) if j > pos - window or j < sinks])
            o, l, s, r = _attention(q[a + i:a + i + 1], k[b + at], v[b + at], [1], [len(at)], scale, False)
            out[a + i], lse[a + i], spread[a + i], reach[a + i] = o[0], l[0], s[0], r[0]
        a, b = a + n_q, b + n_k
    return out, lse, spread, reach
