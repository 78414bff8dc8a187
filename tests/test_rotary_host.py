"""Rotary frequencies on the host: the scalings' ends, the fixed-point turns,
and the settings that are refused."""
import math

import pytest
import torch

from adapterslotsplusplus_amd.rotary import Rotary, frequencies


def test_plain_and_linear():
    f, m = frequencies(8, 10000.0)
    assert m == 1.0 and f == [10000.0 ** (-i / 4) for i in range(4)]
    g, _ = frequencies(8, 10000.0, dict(type="linear", factor=4))
    assert g == [x / 4 for x in f]
    assert frequencies(2)[0] == [1.0] and frequencies(2, scaling=dict(type="ntk", factor=8))[0] == [1.0]


def test_ntk_stretches_the_slowest_pair_by_the_factor():
    f, _ = frequencies(64, 10000.0)
    g, m = frequencies(64, 10000.0, dict(type="ntk", factor=8.0))
    assert m == 1.0 and g[0] == f[0] and math.isclose(f[-1] / g[-1], 8.0, rel_tol=1e-12)


@pytest.mark.parametrize("kind", ["yarn", "bands"])
def test_fast_pairs_stay_and_slow_ones_are_divided(kind):
    f, _ = frequencies(128, 500000.0)
    g, m = frequencies(128, 500000.0, dict(type=kind, factor=8.0, original_length=8192))
    assert g[0] == f[0] and math.isclose(g[-1], f[-1] / 8, rel_tol=1e-12)
    ratio = [a / b for a, b in zip(f, g)]
    assert all(1 - 1e-12 <= r <= 8 + 1e-9 for r in ratio) and all(a <= b + 1e-9 for a, b in zip(ratio, ratio[1:]))
    assert any(1.01 < r < 7.9 for r in ratio)
    assert math.isclose(m, 0.1 * math.log(8) + 1) if kind == "yarn" else m == 1.0
    if kind == "bands":  # linear in the turns over the trained length
        for a, b in zip(f, g):
            keep = min(max((8192 * a / (2 * math.pi) - 1) / 3, 0), 1)
            assert math.isclose(b, a / 8 * (1 - keep) + a * keep, rel_tol=1e-12)


def test_yarn_takes_an_attention_factor():
    assert frequencies(64, scaling=dict(type="yarn", factor=4, original_length=4096, attention_factor=1.5))[1] == 1.5
    assert frequencies(64, scaling=dict(type="yarn", factor=1.0, original_length=4096))[1] == 1.0


def test_turns_are_64_bit_fractions():
    r = Rotary(64, 10000.0, device="cpu")
    f, _ = frequencies(64, 10000.0)
    assert r.turns.dtype == torch.int64 and r.turns.shape == (32,) and r.dim == 64
    for t, x in zip(r.turns.tolist(), f):
        # Half a unit of 2^-64 turns, and the roundings of four double operations.
        assert math.isclose((t % 2 ** 64) / 2.0 ** 64 * 2 * math.pi, x, rel_tol=4 * 2.0 ** -53, abs_tol=2 * math.pi * 2.0 ** -65)


@pytest.mark.parametrize("args", [dict(dim=7), dict(dim=0), dict(dim=8, base=1.0), dict(dim=8, base=math.nan), dict(dim=8, scaling=dict(type="what")),
                                  dict(dim=8, scaling=dict(factor=2.0)), dict(dim=8, scaling=dict(type="linear")),
                                  dict(dim=8, scaling=dict(type="linear", factor=-1.0)), dict(dim=8, scaling=dict(type="yarn", factor=2.0)),
                                  dict(dim=8, scaling=dict(type="bands", factor=2.0, original_length=100, low_freq_factor=4, high_freq_factor=4))], ids=str)
def test_refusals(args):
    with pytest.raises(RuntimeError, match="Rotary"):
        frequencies(**args)


@pytest.mark.parametrize("more", [dict(type="yarn", beta_fast=0), dict(type="yarn", beta_slow=-1), dict(type="yarn", beta_fast=math.nan),
                                  dict(type="yarn", attention_factor=math.nan), dict(type="bands", low_freq_factor=-math.inf),
                                  dict(type="bands", high_freq_factor=math.inf)], ids=str)
def test_numbers_that_scale_nothing_are_refused(more):
    with pytest.raises(RuntimeError, match="Rotary: .* must be a"):
        frequencies(8, scaling=dict(factor=8.0, original_length=4096, **more))


def test_numbers_left_empty_have_their_defaults():
    for kind, names in (("yarn", ("beta_fast", "beta_slow", "attention_factor")), ("bands", ("low_freq_factor", "high_freq_factor"))):
        some = dict(type=kind, factor=8.0, original_length=4096)
        assert frequencies(64, scaling=dict(some, **{n: None for n in names})) == frequencies(64, scaling=some)
