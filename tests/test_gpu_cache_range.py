"""GPU: turned keys past the tensors' type's range in a cache of 8-bit rows.

A finite magnitude past the type's largest counts as that, and what would come
back as an infinity takes 240 times the row's power of two; infinities and NaN
alone become NaN.

Tolerance: half a step of 4 significant bits (2^-4 relative, or half of 2^-9 of
the row's power of two), and twice what fp32 may differ by (the errors of
test_gpu_heads.py), for elements inside the range; the ones past it are exact.
"""
import math

import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from adapterslotsplusplus_amd.rotary import Rotary
from oracle import cache_ops as co
from tests.test_gpu_heads import DTYPES, held, inside, make_pages, turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


def cached(engine, k, positions, rotary, norm=None):
    """The keys as the cache holds them, their powers of two, and read back in their type."""
    T, heads, dim = k.shape
    kp, vp, ks, vs = make_pages(-(-T // 16), 16, heads, dim, k.dtype, True, "tokens")
    slots = torch.arange(T).cuda()
    d = k.cuda()
    engine.rotate_into_cache(None, d, d, positions.cuda(), rotary, kp, vp, slots, k_scales=ks, v_scales=vs,
                             k_norm=None if norm is None else norm.cuda())
    back, _ = engine.read_cache(kp, vp, slots, k_scales=ks, v_scales=vs, dtype=k.dtype)
    return held(kp, ks).reshape(-1, heads, dim)[:T], ks.cpu().reshape(-1, heads)[:T].long() - 127, back.cpu()


@DTYPES
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 64, False), (128, 128, True), (64, 20, False), (80, 10, True), (128, 32, False)], ids=str)
def test_turned_keys_past_the_range(engine, dim, rot, interleaved, dtype):
    big = torch.finfo(dtype).max
    bits = dict(type="yarn", factor=8.0, original_length=4096) if dtype == torch.float16 else None
    k = torch.full((40, 2, dim), 3.0, dtype=dtype)
    a, b = (0, 1) if interleaved else (0, rot // 2)
    # fp32 must hold the sums: bf16's own range ends where that of fp32 does.
    most = 60000.0 if dtype == torch.float16 else big * 0.70703125
    k[:, 0, a], k[:, 0, b] = most, most
    k[:, 1, a], k[:, 1, b] = -most, most / 2
    at = torch.arange(40)
    got, e, back = cached(engine, k, at, Rotary(rot, 1e4, interleaved, bits, device="cuda"))
    y, err = turned(k, None, 1e-6, at, rot, 1e4, bits, interleaved)
    past = y.abs() > big
    assert dtype == torch.bfloat16 or past.any()
    s = torch.exp2(e.double())[..., None]
    assert got.isfinite().all() and back.isfinite().all() and torch.equal(back.double(), got)
    assert (y.abs().clamp(max=big).amax(-1) <= 448 * s[..., 0] * (1 + 2.0 ** -16)).all()
    assert torch.equal(got[past], (torch.sign(y) * 240 * s)[past])
    top = torch.where(s * 448 > big, s * 240, s * 448)
    want = torch.where(past, got, torch.minimum(y.abs(), top) * torch.sign(y))
    inside(got, want, torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) + 2 * err, "k")


def test_normed_keys_far_past_the_range(engine):
    """Rows whose norm weights and factor take them far past fp16's range (bf16's is
    fp32's): their other elements keep their bits."""
    dtype = torch.float16
    k = torch.ones((16, 1, 64), dtype=dtype)
    norm = torch.full((64,), 2.0, dtype=dtype)
    norm[5], norm[40] = 65504.0, -60000.0
    rotary = Rotary(2, device="cuda")  # (the first two elements turn)
    rotary.factor = 1.0
    got, e, back = cached(engine, k, torch.zeros(16, dtype=torch.int64), rotary, norm)
    assert (e == 8).all() and torch.equal(back.double(), got)
    assert (got[..., 5] == 61440).all() and (got[..., 40] == -61440).all() and (got[..., 7] == 2.0).all()
    rotary.factor = 2.0 ** 14  # 2 * 2^14 in the pair, within the range; then past it
    got, e, _ = cached(engine, k, torch.zeros(16, dtype=torch.int64), rotary, norm)
    assert (got[..., :2] == 32768).all()
    rotary.factor = 2.0 ** 30
    got, e, back = cached(engine, k, torch.zeros(16, dtype=torch.int64), rotary, norm)
    assert (e == 8).all() and (got[..., :2] == 61440).all() and (got[..., 7] == 2.0).all() and back.isfinite().all()


@DTYPES
def test_infinities_and_nan_of_turned_keys(engine, dtype):
    k = torch.full((16, 1, 64), 1.0, dtype=dtype)
    k[3, 0, 2], k[4, 0, 40], k[5, 0, 34] = math.inf, math.nan, -math.inf
    got, _, back = cached(engine, k, torch.ones(16, dtype=torch.int64), Rotary(64, device="cuda"))
    bad = torch.zeros(16, 1, 64, dtype=torch.bool)
    for t, d in ((3, 2), (4, 8), (5, 2)):
        bad[t, 0, d] = bad[t, 0, d + 32] = True
    assert torch.equal(got.isnan(), bad) and torch.equal(back.isnan(), bad) and not got.isinf().any()
    keep = torch.ones(16, dtype=torch.bool)
    keep[3:6] = False
    y = co.rotate(k, torch.ones(16), [1e4 ** (-i / 32) for i in range(32)])
    assert ((got - y).abs()[keep] <= (y.abs() * 2.0 ** -4 + 1e-4)[keep]).all()
