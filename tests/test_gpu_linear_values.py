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


@pytest.mark.parametrize("T", [2, 20, 160])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_gelu_in_the_tail(engine, T, dtype):
    """gelu of every 16-bit value between -13 and 8, within its own size: half
    a unit of the type, 2^-17 of the polynomial and the hardware's functions,
    and six roundings (of v / sqrt 2 twice, squared, of the square, of log2 e and
    its product) of the exponent v^2 / 2."""
    u, least = (2.0 ** -8, 2.0 ** -126) if dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -25)
    all16 = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    values = all16[torch.isfinite(all16) & (all16 >= -13) & (all16 <= 8)]
    announce(f"linear gelu of {len(values)} values T={T} {dtype}")
    x, w = torch.zeros(T, 8, dtype=dtype), torch.zeros(len(values), 8, dtype=dtype)
    x[:, 0], w[:, 0] = 1, values
    got = engine.linear(x.cuda(), w.cuda(), activation="gelu").cpu()
    assert torch.equal(got, got[:1].expand_as(got))
    v = values.double()
    want = 0.5 * v * torch.special.erfc(-v / math.sqrt(2))  # erfc keeps the tail's digits
    bad = (got[0].double() - want).abs() > want.abs() * (u + 2.0 ** -17 + 6 * 2.0 ** -24 * v.square() / 2) + least
    assert not bad.any(), f"gelu({v[bad][0].item()}): {got[0][bad][0].item()}, not {want[bad][0].item()}"
