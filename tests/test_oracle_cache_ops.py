"""The cache's 64-bit definitions against themselves said another way."""
import math

import torch

from oracle import cache_ops as co
from oracle import model_ops as mo
from tests.helpers import gen, randn


def test_e4m3_is_the_types_rounding():
    x = torch.cat([torch.linspace(-460, 460, 5001), torch.randn(4000, generator=gen(0)) * 0.02, torch.arange(0, 64) * 2.0 ** -11])
    assert torch.equal(co.e4m3(x.double()), x.to(torch.float8_e4m3fn).double())


def test_quantised_rows_are_within_half_a_step():
    x = randn((50, 3, 32), 1, torch.float32, 10.0).double()
    v, e = co.quantise(x, 1e38)
    s = torch.exp2(e.double())
    top = x.abs().amax(-1)
    assert (top <= 448 * s).all() and (top > 224 * s).all()
    assert ((v - x).abs() <= torch.maximum(x.abs() / 16, s[..., None] * 2.0 ** -10)).all()
    v, e = co.quantise(torch.tensor([[0.0, 0.0], [math.inf, 1.0], [65504.0, 3.0]]), 65504.0)
    assert e[0] == -126 and torch.isnan(v[1, 0]) and v[1, 1] == 1 and v[2, 0] == 61440


def test_rotation_turns_pairs():
    x = randn((6, 2, 12), 1, torch.float64)
    pos = torch.tensor([0, 1, 5, 100, -7, 3])
    f = [1.0, 0.1, 0.01]
    for interleaved in (False, True):
        y = co.rotate(x, pos, f, 1.0, interleaved)
        assert torch.equal(y[..., 6:], x[..., 6:]) and torch.allclose(y[0], x[0])
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1))
        assert torch.allclose(co.rotate(y, -pos, f, 1.0, interleaved), x)
        # Products of turned rows go by the distance of their positions.
        a, b = co.rotate(x, pos, f, 1.0, interleaved), co.rotate(x, pos + 11, f, 1.0, interleaved)
        assert torch.allclose((a[2] * a[3]).sum(-1), (b[2] * b[3]).sum(-1))


def test_paged_attention_is_attention_over_the_gathered_rows():
    lens_q, lens_k = [3, 1, 0, 2], [20, 1, 5, 33]
    k, v = randn((8, 16, 2, 8), 1, torch.float64), randn((8, 16, 2, 8), 2, torch.float64)
    table = torch.tensor([[3, 1, 0], [2, 0, 0], [5, 0, 0], [7, 0, 6]])
    q = randn((6, 4, 8), 3, torch.float64)
    got = co.paged_attention(q, k, v, table, lens_q, lens_k, 0.3)
    rows = [torch.cat([k[p] for p in t])[:n] for t, n in zip(table, lens_k)], [torch.cat([v[p] for p in t])[:n] for t, n in zip(table, lens_k)]
    want = mo.attention(q, torch.cat(rows[0]), torch.cat(rows[1]), lens_q, lens_k, 0.3)
    assert all(torch.allclose(a, b) for a, b in zip(got, want))
    whole = co.paged_attention(q, k, v, table, lens_q, lens_k, 0.3, window=5, sinks=100)
    assert all(torch.allclose(a, b) for a, b in zip(whole, want))
    few = co.paged_attention(q, k, v, table, lens_q, lens_k, 0.3, window=5, sinks=2)
    keys = rows[0][0][[0, 1] + list(range(13, 18))], rows[1][0][[0, 1] + list(range(13, 18))]
    one = mo.attention(q[:1], keys[0], keys[1], [1], [7], 0.3)
    assert torch.allclose(few[0][0], one[0][0])


def test_magnitudes_past_the_range_count_as_its_end():
    big = 65504.0
    x = torch.tensor([[70000.0, 3.0], [-1e9, 3.0], [65504.0, 3.0], [math.inf, 57344.0], [-math.inf, 1e5]], dtype=torch.float64)
    v, e = co.quantise(x, big)
    assert e.tolist() == [8, 8, 8, 7, 8]
    assert v[:3].tolist() == [[61440.0, 3.0], [-61440.0, 3.0], [61440.0, 3.0]]
    assert torch.isnan(v[3:, 0]).all() and v[3:, 1].tolist() == [57344.0, 61440.0]
