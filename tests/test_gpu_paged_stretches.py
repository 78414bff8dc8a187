"""GPU: paged_attention of chunks over caches whose stretches (keys in whole shares
for workgroups of their own) leave little or nothing of a tile beside its own tokens."""
import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from tests.helpers import announce
from tests.test_gpu_model_ops import check
from tests.test_gpu_paged_attention import BF, HF, Case, each_want

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF, 32, 8, 64), (HF, 64, 16, 32)], ids=str)
def test_little_is_left_of_a_stretch(engine, dtype, heads, kv_heads, dim, small):
    lens_k = [16384, 5598, 6990, 12897, 5554, 11861, 289, 1775, 12945, 3805, 10850, 410, 1801, 714, 2457, 2785]
    for more in (0, 150):  # two further places of the stretches' ends
        keys = [n + more for n in lens_k]
        announce(f"paged stretches {heads}/{kv_heads}x{dim} {dtype} small={small} +{more}")
        c = Case([128] * 16, keys, heads, kv_heads, dim, dtype, page=32, small=small)
        got, lse = c.run(engine)
        want = each_want(c)
        tol, lse_tol = c.tolerance(*want)
        check(got, want[0], tol, "out")
        check(lse, want[1], lse_tol, "lse")
        again = c.run(engine)
        assert torch.equal(got, again[0]) and torch.equal(lse, again[1])
    assert engine.device_errors() == 0
