"""GPU: paged_attention's table entries for keys that no query sees (pages that
were given up behind a window) are neither read nor flagged."""
import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from tests.helpers import announce
from tests.test_gpu_paged_attention import BF, FORM, HF, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


def given_up(c, window, sinks):
    """Which table entries no query sees a key of."""
    out = torch.ones(c.table.shape, dtype=torch.bool)
    for b, (n_q, n_k) in enumerate(zip(c.lens_q, c.lens_k)):
        low = max(0, n_k - n_q + 1 - window)
        for j in range(out.size(1)):
            a, e = j * c.page, min((j + 1) * c.page, n_k)
            if n_q and a < e and (e > low or a < sinks):
                out[b, j] = False
    return out


LENS = [([1], [500]), ([1, 4, 0, 2], [500, 777, 300, 64]), ([5] * 30, list(range(20, 1520, 50))), ([200], [900]), ([130, 1, 400], [700, 650, 400]), ([9, 3], [4, 900])]


@pytest.mark.parametrize("lens_q,lens_k", LENS, ids=lambda v: str(v)[:20])
@FORM
def test_pages_out_of_sight_need_not_be_there(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, kw):
    announce(f"paged sight q={str(lens_q)[:40]} k={str(lens_k)[:40]} {heads}/{kv_heads}x{dim} {dtype} {kw}")
    for window, sinks in ((1, 0), (16, 0), (16, 3), (40, 20), (100, 130), (3, 300)):
        c = Case(lens_q, lens_k, heads, kv_heads, dim, dtype, **kw)
        want, lse = c.run(engine, window=window, sinks=sinks)
        good, gone = c.table, given_up(c, window, sinks)
        engine.device_errors()
        for bad in (-1, 2 ** 30):
            c.table = torch.where(gone, torch.tensor(bad, dtype=torch.int32), good)
            got, got_lse = c.run(engine, window=window, sinks=sinks)
            assert torch.equal(got, want) and torch.equal(got_lse, lse)
            assert engine.device_errors() == 0, (window, sinks, bad)


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
def test_long_walks_behind_a_window(engine, small):
    """Row tiles of more steps than are listed at a time, their first keys in the middle of a step."""
    c = Case([600], [9000], 64, 32, 64, HF, page=32, small=small)
    for window, sinks in ((4960, 0), (4960, 300), (4999, 33)):
        want, lse = c.run(engine, window=window, sinks=sinks)
        good = c.table
        c.table = torch.where(given_up(c, window, sinks), torch.tensor(-1, dtype=torch.int32), good)
        engine.device_errors()
        got, got_lse = c.run(engine, window=window, sinks=sinks)
        c.table = good
        assert torch.equal(got, want) and torch.equal(got_lse, lse)
        assert engine.device_errors() == 0, (window, sinks)


def test_a_seen_page_outside_the_cache_is_still_flagged(engine):
    for lens_q, lens_k in (([1], [500]), ([200], [700])):
        c = Case(lens_q, lens_k, 4, 2, 64, BF)
        low = lens_k[0] - lens_q[0] + 1 - 20
        for window, sinks, page in ((20, 0, low // 16), (20, 0, (lens_k[0] - 1) // 16), (20, 17, 1)):
            good = c.table.clone()
            c.table[0, page] = -1
            engine.device_errors()
            c.run(engine, window=window, sinks=sinks)
            assert engine.device_errors() == 1, (window, sinks, page)
            c.table = good
