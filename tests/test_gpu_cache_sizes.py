"""GPU: more rows of heads than one launch takes (a grid has fewer than 2^32
threads, and a token takes a wave of 64 or more)."""
import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from adapterslotsplusplus_amd.rotary import Rotary
from tests.helpers import announce

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


@pytest.mark.parametrize("dim,rot", [(16, 16), (8, 8)], ids=["pairs", "rows"])
def test_many_tokens_rotate(engine, dim, rot):
    T, cut = (1 << 26) + 77, (1 << 25) + 5
    announce(f"rotate {T} tokens of 1x{dim}")
    x = torch.empty(T, 1, dim, dtype=BF, device="cuda").normal_()
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 37
    rotary = Rotary(rot, device="cuda")
    got, none = engine.rotate_heads(x, None, pos, rotary)
    assert none is None
    for a in range(0, T, cut // 3):
        part = slice(a, min(T, a + cut // 3))
        assert torch.equal(got[part], engine.rotate_heads(x[part], None, pos[part], rotary)[0])
    engine.rotate_heads(x, None, pos, rotary, q_out=x)
    assert torch.equal(x, got)


@pytest.mark.parametrize("small", [False, True], ids=["same", "e4m3"])
def test_many_tokens_through_a_cache(engine, small):
    T, dim, page = (1 << 26) + 77, 16, 1 << 12
    announce(f"cache {T} tokens of 1x{dim} small={small}")
    pages = -(-T // page)
    kind = torch.float8_e4m3fn if small else BF
    kp, vp = (torch.empty(pages, page, 1, dim, dtype=torch.uint8 if small else BF, device="cuda") for _ in range(2))
    kp, vp = kp.view(kind), vp.view(kind)
    scales = {n: torch.empty(pages, page, 1, dtype=torch.uint8, device="cuda") for n in ("k_scales", "v_scales")} if small else {}
    # Rows that either cache holds exactly: four bits and a power of two.
    k = torch.randint(-8, 9, (T, 1, dim), dtype=torch.int8, device="cuda").to(BF)
    v = k.flip(0)
    slots = T - 1 - torch.arange(T, device="cuda", dtype=torch.int32)
    engine.device_errors()
    engine.write_cache(k, v, kp, vp, slots, **scales)
    a, b = engine.read_cache(kp, vp, slots, dtype=BF, **scales)
    assert torch.equal(a, k) and torch.equal(b, v)
    turned = engine.rotate_into_cache(k, k, v, slots, None, kp, vp, slots, **scales)
    assert torch.equal(turned, k)
    a, b = engine.read_cache(kp, vp, slots[:1000], dtype=BF, **scales)
    assert torch.equal(a, k[:1000]) and torch.equal(b, v[:1000])
    assert engine.device_errors() == 0
