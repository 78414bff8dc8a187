"""GPU: paged_attention over the longest cache that a length can name.

Keys are zero and values one, so that every weight is one: a share of 2^22 keys is
summed exactly, the 512 shares' sum is off by at most 2^9 * 2^-24 of itself, and so
is what the outputs are divided by."""
import math

import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from tests.helpers import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
@pytest.mark.parametrize("tokens", [40, 1], ids=["tile", "chunk"])
def test_lengths_up_to_31_bits(engine, tokens, small):
    """One page named 128 times; table entries beside the request's name none."""
    page, dim = 1 << 24, 16 if small else 8
    announce(f"paged longest, {tokens} tokens, small={small}")
    if small:
        k = torch.zeros(1, page, 1, dim, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        v = torch.full((1, page, 1, dim), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        s = torch.full((1, page, 1), 127, dtype=torch.uint8, device="cuda")
        scales = dict(k_scales=s, v_scales=s)
    else:
        k, v = (torch.full((1, page, 1, dim), x, dtype=torch.bfloat16, device="cuda") for x in (0.0, 1.0))
        scales = {}
    tables = torch.full((4096,), -1, dtype=torch.int32, device="cuda")
    table = tables[2048:2176].view(1, 128)
    table.zero_()
    q = torch.ones(tokens, 1, dim, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    engine.device_errors()
    for given, n in ((2 ** 31 - 1, 2 ** 31 - 256), (2 ** 31 - 300, 2 ** 31 - 300)):
        kv = torch.tensor([given], dtype=torch.int32, device="cuda")
        out, lse = engine.paged_attention(q, k, v, table, cu, kv, return_lse=True, **scales)
        assert engine.device_errors() == 0
        assert (out == 1).all()
        assert ((lse.double() - math.log(n)).abs() <= 2.0 ** -14).all()


def test_more_row_tiles_than_a_grid_holds(engine):
    """2^20 tokens of 2048 heads, each its own key head's: 2^24 row tiles, which
    a grid of a workgroup each would not hold.  All but the last 16 tokens stand
    before the first key."""
    T, heads, dim = 1 << 20, 2048, 8
    announce(f"paged {T} tokens of {heads} heads")
    q = torch.ones(1, heads, dim, dtype=torch.bfloat16, device="cuda").expand(T, heads, dim)
    k, v = (torch.full((1, 16, heads, dim), x, dtype=torch.bfloat16, device="cuda") for x in (0.0, 1.0))
    out = torch.full((T, heads, dim), 3.0, dtype=torch.bfloat16, device="cuda")
    cu, kv = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, T], [16]))
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    engine.paged_attention(q, k, v, table, cu, kv, out=out)
    assert (out[-16:] == 1).all()
    for part in out[:-16].split(1 << 16):
        assert (part == 0).all()
