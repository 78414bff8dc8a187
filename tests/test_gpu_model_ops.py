"""GPU: linear, packed_attention and token_logprobs against their 64-bit
definitions (oracle/model_ops.py), at the sizes, strides and masks where they
can go wrong.

Tolerances are the errors an evaluation in fp32 with one rounding to the
tensors' type may have:
  * u(type) = 2^-8 (bf16), 2^-11 (fp16): half a unit in the last place,
    relative; 2^-25 absolute below fp16's normal range;
  * an fp32 sum of n terms in any order: n * 2^-23 * sum of magnitudes (2^-24
    a step, and as much again for the matrix cores' own alignment).
"""
import math

import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from oracle import model_ops as mo
from tests.helpers import announce, gen, randn

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


def check(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    bad = ~((got - want).abs() <= tol) & (got != want)
    if bad.any():
        i = int(torch.nonzero(bad.flatten())[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: got "
                             f"{got.flatten()[i].item():.7g}, want {want.flatten()[i].item():.7g}, may differ by "
                             f"{tol.expand_as(want).flatten()[i].item():.3g}")


# ------------------------------------------------------------------- linear --

def linear_tol(y, size, d_in, dtype):
    # The activations' slopes stay under 1.13, their own evaluation within
    # 2^-18 of the magnitudes involved.
    t = 1.13 * (d_in + 4) * 2.0 ** -23 * size + 2.0 ** -18 * (1 + size.clamp_max(16))
    return t + U[dtype] * (y.abs() + t) + 2.0 ** -25


def linear_case(engine, T, d_in, n, dtype, act="none", gated=False, bias=False, residual=False, seed=0, layout="plain"):
    announce(f"linear T={T} d_in={d_in} n={n} {dtype} {act} gated={gated} bias={bias} residual={residual} {layout}")
    rows = 2 * n if gated else n
    x, w = randn((T, d_in), seed, dtype), randn((rows, d_in), seed + 1, dtype, max(d_in, 1) ** -0.5)
    b = randn((rows,), seed + 2, dtype) if bias else None
    r = randn((T, n), seed + 3, dtype) if residual else None
    want, size = mo.linear(x, w, b, r, act, gated)

    def place(t, pad, shift):
        """t on the device inside a larger buffer of NaN."""
        if t is None or layout == "plain":
            return None if t is None else t.cuda()
        buf = torch.full((t.size(0) * (t.size(1) + pad) + 64,), float("nan"), dtype=dtype, device="cuda")
        view = buf[shift:shift + t.size(0) * (t.size(1) + pad)].view(t.size(0), -1)[:, :t.size(1)]
        view.copy_(t)
        return view

    pad, shift = {"plain": (0, 0), "padded": (8, 16), "odd": (3, 1)}[layout]
    out = place(torch.zeros(T, n, dtype=dtype), pad, shift)
    y = engine.linear(place(x, pad, shift), place(w, pad, shift), bias=None if b is None else b.cuda(),
                      residual=place(r, pad, shift), activation=act, gated=gated, out=None if layout == "plain" else out)
    check(y, want, linear_tol(want, size, d_in, dtype), "linear")
    if layout != "plain":
        assert y is out
        assert torch.isnan(out._base).sum() == out._base.numel() - T * n, "written outside the output"


SIZES = [(1, 1, 1), (1, 64, 16), (1, 4096, 4096), (1, 520, 77), (2, 7, 5), (3, 8, 130), (7, 264, 1000), (15, 200, 33),
         (16, 128, 64), (17, 72, 257), (31, 1544, 100), (33, 65, 129), (48, 2048, 512), (64, 63, 64), (65, 512, 260),
         (100, 1000, 1101), (127, 96, 31), (128, 2048, 2048), (129, 4096, 144), (200, 64, 4096), (257, 320, 300),
         (300, 1544, 1101), (513, 128, 640), (700, 8, 96), (1025, 200, 264), (130, 8192, 40)]


@pytest.mark.parametrize("T,d_in,n", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_linear_sizes(engine, T, d_in, n, dtype):
    acts = ["none", "relu", "gelu", "gelu_tanh", "silu"]
    k = SIZES.index((T, d_in, n))
    linear_case(engine, T, d_in, n, dtype, acts[k % 5], gated=False, bias=k % 2 == 0, residual=k % 3 == 0, seed=k)
    linear_case(engine, T, d_in, n, dtype, acts[(k + 4) % 5], gated=True, bias=k % 3 == 1, residual=k % 2 == 1, seed=k + 50)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("T", [1, 40, 160])
def test_linear_epilogues(engine, act, T):
    for gated in (False, True):
        for bias in (False, True):
            for residual in (False, True):
                linear_case(engine, T, 136, 84, torch.bfloat16, act, gated, bias, residual, seed=T)


@pytest.mark.parametrize("layout", ["padded", "odd"])
@pytest.mark.parametrize("T,d_in,n", [(1, 256, 64), (5, 100, 33), (20, 72, 48), (70, 129, 65), (150, 512, 200), (300, 264, 270)], ids=str)
def test_linear_layouts(engine, T, d_in, n, layout):
    """Rows apart, pointers at any element, and nothing written between."""
    linear_case(engine, T, d_in, n, torch.bfloat16, "gelu", False, True, True, seed=T, layout=layout)
    linear_case(engine, T, d_in, n, torch.float16, "silu", True, True, True, seed=T + 1, layout=layout)


def test_linear_large_tile_sizes(engine):
    """Sizes of the largest tiles, against fp64 products on the device."""
    for T, d_in, n, gated, dtype in ((512, 1024, 4096, True, torch.bfloat16), (2048, 520, 2100, False, torch.float16),
                                     (1000, 2056, 1500, True, torch.float16), (4100, 576, 2304, False, torch.bfloat16)):
        announce(f"linear large T={T} d_in={d_in} n={n} gated={gated} {dtype}")
        x, w = randn((T, d_in), 1, dtype).cuda(), randn((2 * n if gated else n, d_in), 2, dtype, 0.05).cuda()
        r = randn((T, n), 3, dtype).cuda()
        want, size = mo.linear(x, w, None, r, "silu", gated)
        got = engine.linear(x, w, residual=r, activation="silu", gated=gated)
        check(got, want.cpu(), linear_tol(want, size, d_in, dtype).cpu(), "linear")


def test_linear_rows_do_not_mix(engine):
    """NaN and infinity in one row of x, or of the weight, stay in their row or column."""
    for T in (3, 40, 150, 600):
        x, w = randn((T, 256), 0, torch.bfloat16).cuda(), randn((200, 256), 1, torch.bfloat16).cuda()
        clean = engine.linear(x, w)
        x[1, 5], x[2, 255], w[7, 0] = float("nan"), float("inf"), float("nan")
        y = engine.linear(x, w, activation="relu")
        assert torch.isnan(y[1]).all() and torch.isnan(y[:, 7]).all()
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[1:3] = False
        keep[:, 7] = False
        assert torch.equal(y[keep], torch.relu(clean)[keep])


def test_linear_residual_in_place_and_batch_shapes(engine):
    x, w = randn((2, 9, 64), 0, torch.float16).cuda(), randn((48, 64), 1, torch.float16).cuda()
    r = randn((2, 9, 48), 2, torch.float16).cuda()
    y = engine.linear(x, w, residual=r)
    assert y.shape == (2, 9, 48)
    buf = r.reshape(18, 48).clone()
    assert engine.linear(x, w, residual=buf, out=buf) is buf
    assert torch.equal(buf, y.view(18, 48))
    assert engine.linear(x[:, :0], w).shape == (2, 0, 48)
    one = x[:1, :1].reshape(1, 64).expand(5, 64)  # rows 0 elements apart
    assert torch.equal(engine.linear(one, w), engine.linear(one.contiguous(), w))


def test_linear_no_columns_is_bias_and_residual(engine):
    r = randn((5, 12), 2, torch.bfloat16).cuda()
    x, w = torch.zeros(5, 0, dtype=torch.bfloat16, device="cuda"), torch.zeros(12, 0, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(engine.linear(x, w, residual=r), r)


def test_linear_repeats_bit_for_bit(engine):
    for T, d_in, n in ((1, 4096, 512), (16, 4096, 256), (128, 2048, 512), (100, 8192, 128)):
        x, w = randn((T, d_in), 0, torch.bfloat16).cuda(), randn((n, d_in), 1, torch.bfloat16).cuda()
        first = engine.linear(x, w)
        for _ in range(5):
            assert torch.equal(engine.linear(x, w), first)


def test_linear_refusals(engine):
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 16, dtype=torch.bfloat16, device="cuda")
    for bad, kw in ((lambda: engine.linear(x.float(), w), "fp16 or bf16"), (lambda: engine.linear(x, w.half()), "one dtype"),
                    (lambda: engine.linear(x[:, :8], w), "must be"), (lambda: engine.linear(x, w.t()), "must be"),
                    (lambda: engine.linear(x, w, activation="tanh"), "activation"),
                    (lambda: engine.linear(x, w[:7], gated=True), "as many"), (lambda: engine.linear(x, w[:0]), "no rows"),
                    (lambda: engine.linear(x, w, bias=x[0]), "bias"), (lambda: engine.linear(x, w, residual=x), "residual"),
                    (lambda: engine.linear(x, w, out=x), "out must"), (lambda: engine.linear(x.cpu(), w), "CUDA"),
                    (lambda: engine.linear(x, torch.zeros(16, 16, dtype=torch.bfloat16, device="cuda").t()[:8]), "unit")):
        with pytest.raises(RuntimeError, match=kw):
            bad()


# ---------------------------------------------------------------- attention --

def bounds(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()


def attention_tol(out, lse, spread, reach, dim, lens_k, v_max, dtype):
    u = U[dtype]
    n = max(lens_k) + 8
    score = (dim + 4) * 2.0 ** -23 * reach + 2.0 ** -21  # of a score, and of exp2's argument
    each = (u + 2 * score + n * 2.0 ** -23)[..., None]
    tol = 1.02 * each * spread + u * out.abs() + 2.0 ** -25
    if dtype == torch.float16:  # exponentials below fp16's normal range
        tol = tol + n * 2.0 ** -25 * v_max
    return tol, score + n * 2.0 ** -23 + 2.0 ** -22 * lse.abs().nan_to_num(0, 0, 0)


def attention_case(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, causal=True, window=0, scale=None, seed=0,
                   layout="separate", extra=0):
    announce(f"attention q={lens_q} k={lens_k} heads={heads}/{kv_heads}x{dim} {dtype} causal={causal} window={window} {layout}")
    T, S = sum(lens_q), sum(lens_k)
    q, k, v = randn((T, heads, dim), seed, dtype), randn((S, kv_heads, dim), seed + 1, dtype), randn((S, kv_heads, dim), seed + 2, dtype)
    sc = dim ** -0.5 if scale is None else scale
    out, lse, spread, reach = mo.attention(q, k, v, lens_q, lens_k, sc, causal, window)
    if layout == "packed":  # one projection's output, NaN between what is read
        buf = torch.full((T + extra, heads + 2 * kv_heads + 1, dim + 8), float("nan"), dtype=dtype, device="cuda")
        dq, dk, dv = buf[:T, :heads, :dim], buf[:T, heads:heads + kv_heads, :dim], buf[:T, heads + kv_heads:-1, :dim]
        for d, s in ((dq, q), (dk, k), (dv, v)):
            d.copy_(s)
    else:
        dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
    got, got_lse = engine.packed_attention(dq, dk, dv, bounds(lens_q), None if lens_q is lens_k else bounds(lens_k),
                                           scale=scale, causal=causal, window=window, return_lse=True)
    tol, lse_tol = attention_tol(out, lse, spread, reach, dim, lens_k, float(v.abs().max()) if S else 0.0, dtype)
    check(got, out, tol, "out")
    check(got_lse, lse, lse_tol, "lse")


PROMPTS = [1], [2], [31], [32], [33], [63], [64], [65], [127], [128], [129], [255], [256], [257], [300], [1, 1, 1], [5, 0, 70, 1, 0, 130], [0], [64, 64], [100, 200, 3]


@pytest.mark.parametrize("lens", PROMPTS, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 2, 128, torch.bfloat16), (3, 3, 64, torch.float16), (8, 1, 80, torch.bfloat16)],
                         ids=["4/2x128", "3/3x64", "8/1x80"])
def test_attention_prompts(engine, lens, heads, kv_heads, dim, dtype):
    attention_case(engine, lens, lens, heads, kv_heads, dim, dtype, seed=len(lens) + sum(lens))


CACHED = [([1], [1]), ([1], [17]), ([1], [777]), ([1], [2049]), ([1, 1, 1, 1], [1, 64, 65, 500]), ([4, 2, 0, 5], [40, 700, 9, 5]),
          ([3, 8], [600, 33]), ([40], [300]), ([17, 1, 200], [1000, 1000, 1000]), ([1, 0, 1], [0, 5, 3]), ([9], [4]), ([70, 1], [30, 0]),
          ([2] * 40, list(range(2, 202, 5)))]


@pytest.mark.parametrize("lens_q,lens_k", CACHED, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, torch.bfloat16), (2, 2, 64, torch.float16), (7, 1, 96, torch.float16),
                                                      (32, 1, 64, torch.bfloat16)], ids=["8/2x128", "2/2x64", "7/1x96", "32/1x64"])
def test_attention_cached(engine, lens_q, lens_k, heads, kv_heads, dim, dtype):
    """Few queries at the end of longer caches, more queries than keys (rows
    that see nothing), sequences without queries or without keys."""
    attention_case(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, seed=len(lens_q))


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
@pytest.mark.parametrize("lens_q,lens_k", [([200], [200]), ([1, 1], [500, 3]), ([33, 5], [400, 64])], ids=str)
def test_attention_window(engine, lens_q, lens_k, window):
    attention_case(engine, lens_q, lens_k, 4, 2, 64, torch.bfloat16, window=window)
    attention_case(engine, lens_q, lens_k, 4, 1, 128, torch.float16, window=window)


@pytest.mark.parametrize("lens_q,lens_k", [([150], [150]), ([1, 30], [200, 77]), ([5, 300], [3, 190])], ids=str)
def test_attention_not_causal(engine, lens_q, lens_k):
    attention_case(engine, lens_q, lens_k, 4, 2, 128, torch.bfloat16, causal=False)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 56, 72, 88, 104, 112, 120])
def test_attention_head_sizes(engine, dim):
    attention_case(engine, [90, 3], [90, 3], 2, 1, dim, torch.bfloat16, seed=dim)
    attention_case(engine, [1, 2], [300, 70], 4, 2, dim, torch.float16, seed=dim)


@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (4, 1, 128)], ids=str)
@pytest.mark.parametrize("window", [0, 40])
def test_attention_one_longer_among_single_tokens(engine, heads, kv_heads, dim, window):
    # One sequence of several 128-row blocks next to many of a row or two.
    n = 40
    lens_q = [1 + b % 2 for b in range(n)]
    lens_k = [3 * b + 2 for b in range(n)]
    lens_q[7], lens_k[7] = 200, 700
    attention_case(engine, lens_q, lens_k, heads, kv_heads, dim, torch.bfloat16, window=window)


def test_attention_longer_one_among_many_heads(engine):
    # As above with more partial results than the scratch holds: its keys are not split.
    lens_q, lens_k = [1] * 100, [b % 13 + 1 for b in range(100)]
    lens_q[50], lens_k[50] = 40, 700
    attention_case(engine, lens_q, lens_k, 32, 8, 128, torch.float16)


def test_attention_packed_views(engine):
    lens = [60, 1, 90, 130]
    for heads, kv_heads, dim, dtype in ((4, 2, 128, torch.bfloat16), (2, 2, 64, torch.float16), (6, 1, 40, torch.bfloat16)):
        attention_case(engine, lens, lens, heads, kv_heads, dim, dtype, layout="packed", extra=3)
        attention_case(engine, [1, 2], [1, 2], heads, kv_heads, dim, dtype, layout="packed")


def test_attention_scales(engine):
    """Scores that swing far between keys: the running maximum rises in steps."""
    for scale in (0.0, 1.0, 4.0):
        attention_case(engine, [300], [300], 2, 2, 64, torch.bfloat16, scale=scale)
        attention_case(engine, [2], [900], 4, 1, 128, torch.float16, scale=scale)
    T, dim = 400, 64
    k = torch.zeros(T, 1, dim, dtype=torch.float16)
    k[:, 0, 0] = torch.linspace(-60, 60, T)  # each key beats the ones before it
    q = torch.ones(T, 1, dim, dtype=torch.float16)
    v = randn((T, 1, dim), 5, torch.float16)
    for flip in (False, True):
        kk = k.flip(0) if flip else k
        out, lse, spread, reach = mo.attention(q, kk, v, [T], [T], 1.0)
        got, got_lse = engine.packed_attention(q.cuda(), kk.cuda(), v.cuda(), bounds([T]), scale=1.0, return_lse=True)
        tol, lse_tol = attention_tol(out, lse, spread, reach, dim, [T], float(v.abs().max()), torch.float16)
        check(got, out, tol, "out")
        check(got_lse, lse, lse_tol, "lse")


def test_attention_lowest_scores_and_infinite_keys(engine):
    """Keys of the type's lowest values (scores near the fp32 range's end), and
    keys whose scores are -inf: they weigh nothing, and a row of them alone is NaN."""
    dim, T = 64, 130
    q = torch.ones(T, 1, dim, dtype=torch.bfloat16)
    k = randn((T, 1, dim), 0, torch.bfloat16)
    v = randn((T, 1, dim), 1, torch.bfloat16)
    k[10:100] = 0
    k[10:100, 0, 0] = -torch.finfo(torch.bfloat16).max
    k[100, 0, 3] = -math.inf
    out, lse, spread, reach = mo.attention(q, k, v, [T], [T], 0.125)
    got, got_lse = engine.packed_attention(q.cuda(), k.cuda(), v.cuda(), bounds([T]), return_lse=True)
    tol, lse_tol = attention_tol(out, lse, spread, reach, dim, [T], float(v.abs().max()), torch.bfloat16)
    tol, lse_tol = tol.nan_to_num(0.02, 0.02).clamp_max(0.02), lse_tol.nan_to_num(1e-4, 1e-4).clamp_max(1e-4)
    check(got, out, tol, "out")
    check(got_lse, lse, lse_tol, "lse")
    k[:] = 0
    k[:, 0, 3] = -math.inf
    got, got_lse = engine.packed_attention(q.cuda(), k.cuda(), v.cuda(), bounds([T]), return_lse=True)
    assert torch.isnan(got).all()


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1)])
def test_attention_unseen_keys_do_not_matter(engine, heads, kv_heads):
    """NaN and infinity in keys and values that a query does not see (later
    ones, earlier than its window, other sequences' ones) leave it as it is."""
    lens_q, lens_k = [100, 2, 150], [100, 300, 150]
    T, S = sum(lens_q), sum(lens_k)
    q, k, v = (randn((n, h, 64), i, torch.bfloat16).cuda() for i, (n, h) in enumerate(((T, heads), (S, kv_heads), (S, kv_heads))))
    cu_q, cu_k = bounds(lens_q), bounds(lens_k)
    for window in (0, 40):
        clean = engine.packed_attention(q, k, v, cu_q, cu_k, window=window)
        for at in (0, 99, 100, 399, 400, 470, 549):
            b = 0 if at < 100 else 1 if at < 400 else 2
            at_q, at_k = sum(lens_q[:b]), sum(lens_k[:b])
            pos = torch.arange(lens_q[b]) + lens_k[b] - lens_q[b]
            sees = (pos >= at - at_k) & ((pos - window < at - at_k) if window else True)
            seen = torch.zeros(T, dtype=torch.bool)
            seen[at_q:at_q + lens_q[b]] = sees
            for value in (math.nan, math.inf, -math.inf):
                k2, v2 = k.clone(), v.clone()
                v2[at] = value
                got = engine.packed_attention(q, k, v2, cu_q, cu_k, window=window)
                assert torch.equal(got[~seen], clean[~seen]), f"v[{at}] = {value}, window {window}"
                assert not torch.isfinite(got[seen]).any(), f"v[{at}] = {value}, window {window}: lost"
                k2[at] = math.nan
                got = engine.packed_attention(q, k2, v, cu_q, cu_k, window=window)
                assert torch.equal(got[~seen], clean[~seen]), f"k[{at}] = nan, window {window}"
                assert torch.isnan(got[seen]).all()


def test_attention_rows_of_no_sequence(engine):
    """Rows past the last bound (a padded batch) get 0 and -inf; a batch of no sequences too."""
    q, k = randn((50, 2, 64), 0, torch.float16).cuda(), randn((40, 2, 64), 1, torch.float16).cuda()
    cu = bounds([20, 10])
    out, lse = engine.packed_attention(q, k, k, cu, cu, return_lse=True)
    assert (out[30:] == 0).all() and (lse[30:] == -math.inf).all()
    assert torch.equal(out[:30], engine.packed_attention(q[:30], k[:30], k[:30], cu))
    out, lse = engine.packed_attention(q, k, k, bounds([]), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out = engine.packed_attention(q, k[:0], k[:0], bounds([50]), bounds([0]))
    assert (out == 0).all()
    assert engine.packed_attention(q[:0], k, k, bounds([0]), bounds([40])).shape == (0, 2, 64)
    # Bounds past the tensors' rows are cut to them.
    over = engine.packed_attention(q, k, k, bounds([60]), bounds([45]))
    assert torch.isfinite(over).all()


def test_attention_out_given(engine):
    lens = [33, 40]
    q, k, v = (randn((73, 4, 64), i, torch.bfloat16).cuda() for i in range(3))
    want = engine.packed_attention(q, k, v, bounds(lens))
    wide = torch.full((73, 5, 72), 7.0, dtype=torch.bfloat16, device="cuda")
    view = wide[:, :4, :64]
    assert engine.packed_attention(q, k, v, bounds(lens), out=view) is view
    assert torch.equal(view, want) and (wide[:, 4] == 7).all() and (wide[:, :, 64:] == 7).all()


def test_attention_offsets_past_32_bits(engine):
    """A cache whose rows lie 64 KiB apart, read past 4 GiB."""
    n, far = 80000, 1 << 15
    store = torch.empty(n * far, dtype=torch.bfloat16, device="cuda")
    k, v = store.view(n, far)[:, :64].unsqueeze(1), store.view(n, far)[:, 64:128].unsqueeze(1)
    lens_k = [n - 300, 300]
    k[-300:], v[-300:] = randn((300, 1, 64), 0, torch.bfloat16).cuda(), randn((300, 1, 64), 1, torch.bfloat16).cuda()
    k[:-300], v[:-300] = 0, 1
    q = randn((3, 4, 64), 2, torch.bfloat16).cuda()
    got = engine.packed_attention(q, k, v, bounds([1, 2]), bounds(lens_k))
    assert (got[0] - 1).abs().max() <= 2.0 ** -8
    want = engine.packed_attention(q[1:], k[-300:].contiguous(), v[-300:].contiguous(), bounds([2]), bounds([300]))
    check(got[1:], want.double().cpu(), torch.tensor(2.0 ** -6), "the far sequence")


def test_attention_longer_prompts(engine):
    """Several tiles of keys and queries, against fp64 on the device."""
    for lens_q, lens_k, heads, kv_heads, dim, dtype, window in (
            ([1500, 600], [1500, 600], 4, 1, 128, torch.bfloat16, 0), ([2000], [2000], 2, 2, 64, torch.float16, 300),
            ([500], [3500], 6, 2, 96, torch.bfloat16, 0), ([1, 3], [20000, 9000], 8, 2, 128, torch.float16, 0)):
        announce(f"attention long {lens_q} {lens_k} {heads}/{kv_heads}x{dim} {dtype} window={window}")
        q = randn((sum(lens_q), heads, dim), 0, dtype).cuda()
        k, v = (randn((sum(lens_k), kv_heads, dim), i, dtype).cuda() for i in (1, 2))
        got, got_lse = engine.packed_attention(q, k, v, bounds(lens_q), bounds(lens_k), window=window, return_lse=True)
        a = b = 0
        for n_q, n_k in zip(lens_q, lens_k):
            qq, kk, vv = q[a:a + n_q].double(), k[b:b + n_k].double(), v[b:b + n_k].double()
            pos = torch.arange(n_q, device="cuda")[:, None] + n_k - n_q
            at = torch.arange(n_k, device="cuda")[None]
            hide = (at > pos) | ((at <= pos - window) if window else torch.zeros_like(at > pos))
            for h in range(heads):
                kh, vh = kk[:, h * kv_heads // heads], vv[:, h * kv_heads // heads]
                s = (qq[:, h] @ kh.t().contiguous()) * dim ** -0.5
                p = torch.softmax(s.masked_fill(hide, -math.inf), 1)
                reach = (qq[:, h].abs() @ kh.abs().t().contiguous()).amax(1) * dim ** -0.5
                lse = torch.logsumexp(s.masked_fill(hide, -math.inf), 1)
                tol, lse_tol = attention_tol(p @ vh, lse, p @ vh.abs(), reach, dim, [n_k], float(vh.abs().max()), dtype)
                check(got[a:a + n_q, h], (p @ vh).cpu(), tol.cpu(), f"out of head {h}")
                check(got_lse[a:a + n_q, h], lse.cpu(), lse_tol.cpu(), f"lse of head {h}")
            a, b = a + n_q, b + n_k


def test_attention_repeats_bit_for_bit(engine):
    q, k, v = (randn((n, h, 128), i, torch.bfloat16).cuda() for i, (n, h) in enumerate(((5, 8), (9000, 2), (9000, 2))))
    cu_q, cu_k = bounds([1, 4]), bounds([2000, 7000])
    first = engine.packed_attention(q, k, v, cu_q, cu_k)
    for _ in range(5):
        assert torch.equal(engine.packed_attention(q, k, v, cu_q, cu_k), first)


def test_attention_refusals(engine):
    q, k = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu = bounds([4])
    f = engine.packed_attention
    wide = torch.zeros(4, 4, 136, dtype=torch.bfloat16, device="cuda")
    odd = torch.zeros(4 * 4 * 65 + 1, dtype=torch.bfloat16, device="cuda")
    for bad, kw in ((lambda: f(q.float(), k, k, cu), "fp16 or bf16"), (lambda: f(q, k.half(), k, cu), "one dtype"),
                    (lambda: f(q, k, k[:3], cu), "must be"), (lambda: f(q[:, :3], k, k, cu), "evenly"),
                    (lambda: f(q[:, :, :60], k[:, :, :60], k[:, :, :60], cu), "head size"),
                    (lambda: f(wide, wide, wide, cu), "head size"), (lambda: f(q, k, k, cu.long()), "int32"),
                    (lambda: f(q, k, k, cu, bounds([2, 2])), "one length"), (lambda: f(q, k, k, cu, causal=False, window=4), "window"),
                    (lambda: f(q, k, k, cu, window=-1), "window"), (lambda: f(q.cpu(), k, k, cu), "CUDA"),
                    (lambda: f(odd[1:1 + 1024].view(4, 4, 64), k, k, cu), "aligned"),
                    (lambda: f(odd[:1040].view(4, 4, 65)[:, :, :64], k, k, cu), "multiples of 8"),
                    (lambda: f(q.transpose(1, 2), k, k, cu), "must be"), (lambda: f(q, k, k, cu, out=k), "out must")):
        with pytest.raises(RuntimeError, match=kw):
            bad()


def test_attention_refuses_rows_past_31_bits(engine):
    row = torch.zeros(1, 1, 8, dtype=torch.bfloat16, device="cuda")
    q = row.expand(65536, 65535, 8)
    with pytest.raises(RuntimeError, match="2.31 rows"):
        engine.packed_attention(q, row, row, bounds([4]), bounds([1]), out=q)


# ----------------------------------------------------------------- logprobs --

def logprobs_tol(x, top_value):
    """Of lse: a thread's sum of vocab / 256 terms errs as a random walk, eight
    deviations of it, and the tree behind it, exp2's argument and log by 2^-20."""
    n = x.size(1)
    t = 2.0 ** -24 * 8 * math.sqrt(max(1, n / 256)) + 2.0 ** -20
    return t + 2.0 ** -22 * top_value


def logprobs_case(engine, rows, vocab, top, dtype, std=3.0, seed=0, banned=0.0, ids64=True, pad=0, shift=0):
    announce(f"logprobs rows={rows} vocab={vocab} top={top} {dtype} std={std} banned={banned} pad={pad} shift={shift}")
    x = randn((rows, vocab), seed, torch.float32, std)
    if banned:
        x[:, torch.rand(vocab, generator=gen(seed + 1)) < banned] = -math.inf
        x[:, vocab // 2] = 0.5
    x = x.to(dtype)
    ids = torch.randint(0, vocab, (rows,), generator=gen(seed + 2))
    ids[: rows // 2] = x[: rows // 2].float().argmax(1)
    if rows > 2:
        ids[1] = -1
    lp, ent, ranks, tlp, tid = mo.token_logprobs(x, ids, top)
    buf = torch.full((rows * (vocab + pad) + 64,), float("nan"), dtype=dtype, device="cuda")
    d = buf[shift:shift + rows * (vocab + pad)].view(rows, vocab + pad)[:, :vocab]
    d.copy_(x)
    got = engine.token_logprobs(d, ids.cuda() if ids64 else ids.cuda().int(), top=top)
    assert torch.equal(got.ranks.cpu(), ranks) and torch.equal(got.top_ids.cpu(), tid)
    most = torch.tensor(float(x.double().masked_fill(x == -math.inf, 0).abs().max()))
    tol = logprobs_tol(x, most)
    check(got.logprobs, lp, tol, "logprobs")
    check(got.top_logprobs, tlp, tol, "top_logprobs")
    # The weighted sum errs by its own terms as well: at most log(vocab) of them.
    check(got.entropy, ent, tol * (2 + math.log(vocab)), "entropy")


@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 500, 511, 1000, 2048, 4099, 8193, 32000, 50001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_logprobs_sizes(engine, vocab, dtype):
    for rows, top in ((1, min(vocab, 5)), (3, min(vocab, 64)), (5, 0), (2, 1)):
        logprobs_case(engine, rows, vocab, top, dtype, seed=vocab + rows)


@pytest.mark.parametrize("rows", [1, 2, 17, 300, 1030])
def test_logprobs_rows(engine, rows):
    logprobs_case(engine, rows, 3001, 20, torch.bfloat16, seed=rows)
    logprobs_case(engine, rows, 40000 if rows < 100 else 9000, 7, torch.float32, seed=rows, ids64=False)


def test_logprobs_large_vocabulary(engine):
    for dtype in (torch.float32, torch.bfloat16):
        logprobs_case(engine, 3, 200001, 64, dtype)
        logprobs_case(engine, 70, 128000, 20, dtype, std=1.0)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 5), (8, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_logprobs_layouts(engine, pad, shift, dtype):
    """Rows at any element, NaN between them."""
    logprobs_case(engine, 5, 4001, 10, dtype, pad=pad, shift=shift)
    logprobs_case(engine, 40, 777, 3, dtype, pad=pad, shift=shift)


def test_logprobs_masked(engine):
    for banned in (0.01, 0.5, 0.99, 1.0):
        logprobs_case(engine, 6, 5000, 64, torch.bfloat16, banned=banned)
        logprobs_case(engine, 6, 33000, 20, torch.float32, banned=banned)


@pytest.mark.parametrize("vocab", [300, 20000, 70000])
def test_logprobs_ties_and_orders(engine, vocab):
    """Equal logits rank by id; rising rows make every logit an alternative for a while."""
    for x in (torch.zeros(2, vocab), torch.arange(vocab).float().expand(2, vocab) / vocab,
              -torch.arange(vocab).float().expand(2, vocab) / vocab, (torch.arange(vocab) % 7).float().expand(2, vocab),
              torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0).expand(2, vocab)):
        ids = torch.tensor([vocab - 1, vocab // 3])
        lp, ent, ranks, tlp, tid = mo.token_logprobs(x, ids, 40)
        got = engine.token_logprobs(x.contiguous().cuda(), ids.cuda(), top=40)
        assert torch.equal(got.top_ids.cpu(), tid) and torch.equal(got.ranks.cpu(), ranks)
        tol = logprobs_tol(x, x.abs().max().double())
        check(got.logprobs, lp, tol, "logprobs")
        check(got.entropy, ent, tol * (2 + math.log(vocab)), "entropy")


def test_logprobs_extreme_values(engine):
    """The type's lowest and highest values, rows without a distribution, NaN: each in its own row."""
    for vocab in (1000, 30000):
        x = randn((6, vocab), 0, torch.float32)
        x[0] = torch.finfo(torch.float32).min
        x[1, 5] = torch.finfo(torch.float32).max
        x[2] = -math.inf
        x[3, 77] = math.nan
        x[4, 500] = math.inf
        got = engine.token_logprobs(x.cuda(), torch.tensor([3, 5, 0, 1, 500, 2]).cuda(), top=4)
        assert abs(float(got.logprobs[0]) + math.log(vocab)) < 1e30 and got.top_ids[0].tolist() == [0, 1, 2, 3]
        assert abs(float(got.entropy[0]) - math.log(vocab)) < 1e-4
        assert float(got.logprobs[1]) == 0 and float(got.entropy[1]) == 0 and int(got.ranks[1]) == 1
        assert got.top_logprobs[1, 1:].isfinite().all() or (got.top_logprobs[1, 1:] <= -3e38).all()
        for r in (2, 3, 4):
            assert torch.isnan(got.logprobs[r]) and torch.isnan(got.entropy[r])
        assert got.top_ids[2].tolist() == [0, 1, 2, 3] and int(got.ranks[2]) == 1
        assert int(got.top_ids[3, 0]) == 77 and int(got.top_ids[4, 0]) == 500
        lp, ent, ranks, tlp, tid = mo.token_logprobs(x[5:], torch.tensor([2]), 4)
        assert torch.equal(got.top_ids[5:].cpu(), tid) and torch.equal(got.ranks[5:].cpu(), ranks)
        check(got.logprobs[5:], lp, torch.tensor(1e-5), "the plain row")


def test_logprobs_ids_out_of_range(engine):
    engine.device_errors()
    x = randn((4, 100), 0, torch.float16).cuda()
    got = engine.token_logprobs(x, torch.tensor([-1, 99, -7, 5]).cuda(), top=2)
    assert engine.device_errors() == 0
    assert got.logprobs[0] == 0 and got.ranks[2] == 0 and got.ranks[1] > 0
    got = engine.token_logprobs(x, torch.tensor([100, 1, 2, 1 << 40]).cuda())
    assert engine.device_errors() == 1
    assert got.logprobs[0] == 0 and got.ranks[3] == 0 and got.ranks[1] > 0
    assert got.top_ids.shape == (4, 0)


def test_logprobs_repeats_and_empty(engine):
    x, ids = randn((3, 90000), 0, torch.float32).cuda(), torch.tensor([1, 2, 3]).cuda()
    first = engine.token_logprobs(x, ids, top=9)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(engine.token_logprobs(x, ids, top=9), first))
    got = engine.token_logprobs(x[:0], ids[:0], top=3)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 3)


def test_logprobs_refusals(engine):
    x, ids = torch.zeros(4, 10, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    f = engine.token_logprobs
    for bad, kw in ((lambda: f(x.double(), ids), "fp32"), (lambda: f(x[0], ids), "must be"), (lambda: f(x.t(), ids), "must be"),
                    (lambda: f(x, ids[:3]), "token_ids"), (lambda: f(x, ids.float()), "token_ids"), (lambda: f(x, ids, top=-1), "top"),
                    (lambda: f(x, ids, top=11), "alternatives"), (lambda: f(torch.zeros(4, 100, device="cuda"), ids, top=65), "alternatives"),
                    (lambda: f(x.cpu(), ids), "CUDA"), (lambda: f(x, ids.cpu()), "CUDA"), (lambda: f(x[:, :0], ids), "sizes")):
        with pytest.raises(RuntimeError, match=kw):
            bad()


# ------------------------------------------------------- streams and graphs --

def test_operators_on_another_stream_and_captured(engine):
    """On a side stream, and recorded into a graph that is replayed with new
    inputs between other work, the answers are the eager ones'."""
    T, d = 6, 256
    x, w = randn((T, d), 0, torch.bfloat16).cuda(), randn((d * 3, d), 1, torch.bfloat16, 0.06).cuda()
    head = randn((30000, d), 2, torch.bfloat16).cuda()
    k, v = (randn((900, 2, 64), i, torch.bfloat16).cuda() for i in (3, 4))
    cu_q, cu_k = bounds([1, 5]), bounds([500, 400])
    ids = torch.arange(T, device="cuda")

    def step():
        y = engine.linear(x, w, activation="silu")
        o = engine.packed_attention(y[:, :d].view(T, 4, 64), k, v, cu_q, cu_k)
        h = engine.linear(o.view(T, d), w[:2 * d], residual=x, gated=True)
        logits = engine.linear(h, head)
        return (y, o, h, logits) + tuple(engine.token_logprobs(logits, ids, top=5))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    eager = step()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for seed in range(4):
        x.copy_(randn((T, d), 20 + seed, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in recorded]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {seed}"
