"""The 64-bit oracle of the operators around the apply against torch's own
functions in 64 bits, on the CPU."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import model_ops as mo
from tests.helpers import randn


@pytest.mark.parametrize("act,f", [("none", lambda a: a), ("relu", torch.relu), ("gelu", F.gelu), ("silu", F.silu),
                                   ("gelu_tanh", lambda a: F.gelu(a, approximate="tanh"))])
@pytest.mark.parametrize("gated", [False, True])
def test_linear(act, f, gated):
    x, w, b, r = (randn(s, i, torch.float64) for i, s in enumerate([(5, 24), (14, 24), (14,), (5, 7 if gated else 14)]))
    y, size = mo.linear(x, w, b, r, act, gated)
    a = F.linear(x, w, b)
    want = f(a[:, :7]) * a[:, 7:] + r if gated else f(a) + r
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-12)
    assert (size >= (y - r).abs() * 0.99).all() or act != "none"


@pytest.mark.parametrize("n_q,n_k,window", [(7, 7, 0), (3, 11, 0), (1, 5, 0), (6, 20, 4)])
def test_attention(n_q, n_k, window):
    q, k, v = randn((n_q, 4, 16), 0, torch.float64), randn((n_k, 2, 16), 1, torch.float64), randn((n_k, 2, 16), 2, torch.float64)
    out, lse, _, _ = mo.attention(q, k, v, [n_q], [n_k], 0.25, True, window)
    pos = torch.arange(n_q)[:, None] + n_k - n_q
    seen = torch.arange(n_k)[None] <= pos
    if window:
        seen &= torch.arange(n_k)[None] > pos - window
    kk, vv = (t.repeat_interleave(2, 1).transpose(0, 1) for t in (k, v))
    want = F.scaled_dot_product_attention(q.transpose(0, 1), kk, vv, attn_mask=seen, scale=0.25).transpose(0, 1)
    assert torch.allclose(out, want, rtol=1e-12, atol=1e-12)
    s = (torch.einsum("ihd,hjd->ihj", q, kk) * 0.25).masked_fill(~seen[:, None], -math.inf)
    assert torch.allclose(lse, torch.logsumexp(s, -1), rtol=1e-12)


def test_attention_rows_without_keys_are_empty():
    q, k = randn((4, 1, 8), 0, torch.float64), randn((2, 1, 8), 1, torch.float64)
    out, lse, _, _ = mo.attention(q, k, k, [4, 0], [2, 0], 1.0)
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all()
    assert torch.allclose(out[2], k[0]) and torch.isfinite(lse[2:]).all()


def test_token_logprobs():
    x = randn((6, 50), 0, torch.float64)
    x[:, 7] = x[:, 3]
    x[2, 10:40] = -math.inf
    ids = torch.tensor([0, 3, 5, -1, 50, 49])
    lp, ent, ranks, tlp, tid = mo.token_logprobs(x, ids, 50)
    want = torch.log_softmax(x, 1)
    for i in (0, 1, 2, 5):
        assert torch.allclose(lp[i], want[i, ids[i]]) and ranks[i] == 1 + int((x[i] > x[i, ids[i]]).sum())
    assert lp[3] == 0 and ranks[3] == 0 and lp[4] == 0 and ranks[4] == 0
    for i in range(6):
        assert torch.allclose(ent[i], torch.distributions.Categorical(logits=x[i]).entropy())
        assert tid[i].tolist() == sorted(range(50), key=lambda j: (-float(x[i, j]), j))
    assert torch.allclose(tlp, want.gather(1, tid.long()))
