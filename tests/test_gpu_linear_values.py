"""GPU: linear's activations at values that the random inputs of the other
tests do not reach."""
import math

import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from oracle import model_ops as mo
from tests.helpers import announce

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
# (tokens, outputs) that run on a few tokens' kernel and on tiles.
SIZES = [(2, 8), (40, 48), (160, 4096)]


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


def through(engine, values, act, dtype, T, n):
    """The activation at `values`, as sums of a product: [T, n], value t % len in row t."""
    x = torch.zeros(T, 8, dtype=dtype)
    x[:, 0] = values.to(dtype)[torch.arange(T) % len(values)]
    w = torch.zeros(n, 8, dtype=dtype)
    w[:, 0] = 1
    return engine.linear(x.cuda(), w.cuda(), activation=act).cpu(), x[:, :1]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,n", SIZES, ids=str)
def test_infinity_and_the_largest_values(engine, act, T, n):
    for dtype in (torch.bfloat16, torch.float16):
        most = torch.finfo(dtype).max
        values = torch.tensor([math.inf, most, most / 2, 200.0, -200.0, -most, -math.inf, math.nan])
        announce(f"linear {act} of infinities T={T} n={n} {dtype}")
        got, x = through(engine, values, act, dtype, T, n)
        want = mo.activate(x.double(), act).expand(T, n)
        assert torch.equal(got.double().nan_to_num(7e38), want.to(dtype).double().nan_to_num(7e38))
