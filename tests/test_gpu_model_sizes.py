"""GPU: sizes and strides at the ends of what the operators around the apply take."""
import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from tests.helpers import announce, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


def test_sizes_past_31_bits_are_refused(engine):
    """Not cut to their low 32 bits."""
    announce("operators, sizes past 31 bits")
    far = 2 ** 32 + 8
    x, one = randn((2, 8), 0, torch.bfloat16).cuda(), torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="31 bits"):
        engine.linear(one, one.expand(far, 1))
    with pytest.raises(RuntimeError, match="31 bits"):
        engine.linear(one.expand(1, far), one.expand(1, far))
    ids = torch.zeros(1, dtype=torch.int64, device="cuda")
    for top in (65, 2 ** 32, 2 ** 32 + 1):
        with pytest.raises(RuntimeError, match="alternatives"):
            engine.token_logprobs(x[:1], ids, top=top)
    with pytest.raises(RuntimeError, match="31 bits"):
        engine.token_logprobs(torch.empty(1, far, dtype=torch.float16, device="cuda"), ids)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def test_attention_over_a_head_major_cache(engine):
    """[kv_heads, keys, dim]: heads lie more than 2^22 elements apart."""
    n = 40000
    q = randn((3, 4, 128), 0, torch.bfloat16).cuda()
    k, v = (randn((2, n, 128), i, torch.bfloat16).cuda().permute(1, 0, 2) for i in (1, 2))
    announce(f"attention, head strides {q.stride(1)} {k.stride(1)}")
    got = engine.packed_attention(q, k, v, ints(0, 3), ints(0, n))
    assert torch.equal(got, engine.packed_attention(q, k.contiguous(), v.contiguous(), ints(0, 3), ints(0, n)))
    # Queries and outputs head by head too.
    wide = torch.zeros(4, 40000, 128, dtype=torch.bfloat16, device="cuda").permute(1, 0, 2)
    wide[:3] = q
    out = torch.zeros_like(wide)
    assert out.stride(1) > 1 << 22
    engine.packed_attention(wide[:3], k, v, ints(0, 3), ints(0, n), out=out[:3])
    assert torch.equal(out[:3], got) and not out[3:].any()


def test_attention_keys_far_apart(engine):
    """As far as is taken, and the message past that."""
    far, n = 1 << 24, 70
    store = torch.zeros(n * (far + 8), dtype=torch.bfloat16, device="cuda")
    small = randn((n, 2, 1, 64), 0, torch.bfloat16).cuda()
    q = randn((5, 4, 64), 1, torch.bfloat16).cuda()
    want = engine.packed_attention(q, small[:, 0], small[:, 1], ints(0, 5), ints(0, n))
    for heads in (4, 128):  # key chunks, a row tile
        qh = q[:, :1].expand(5, heads, 64)
        view = store[:n * far].view(n, far)[:, :128].view(n, 2, 1, 64)
        view.copy_(small)
        announce(f"attention, keys {view.stride(0)} apart, {heads} heads")
        assert torch.equal(engine.packed_attention(qh, view[:, 0], view[:, 1], ints(0, 5), ints(0, n)),
                           engine.packed_attention(qh, small[:, 0], small[:, 1], ints(0, 5), ints(0, n)))
    far_q = store[:5 * (far + 8)].view(5, far + 8)[:, :256].view(5, 4, 64)
    far_q.copy_(q)
    assert torch.equal(engine.packed_attention(far_q, small[:, 0], small[:, 1], ints(0, 5), ints(0, n)), want)
    past = store.view(n, far + 8)[:, :64].unsqueeze(1)
    with pytest.raises(RuntimeError, match="16777216 elements apart"):
        engine.packed_attention(q, past, past, ints(0, 5), ints(0, n))


def test_attention_strides_of_one_entry_do_not_matter(engine):
    q, k = randn((1, 2, 64), 0, torch.bfloat16).cuda(), randn((9, 1, 64), 1, torch.bfloat16).cuda()
    want = engine.packed_attention(q, k, k, ints(0, 1), ints(0, 9))
    announce("attention, strides of size-one dimensions")
    odd_q, odd_k = q.as_strided(q.shape, (3, 64, 1)), k.as_strided(k.shape, (64, 1 << 40, 1))
    out = torch.empty_like(q).as_strided(q.shape, (5, 64, 1))
    assert torch.equal(engine.packed_attention(odd_q, odd_k, odd_k, ints(0, 1), ints(0, 9), out=out), want)
    one = k[:1].as_strided((1, 1, 64), (1, 1, 1))
    assert torch.equal(engine.packed_attention(odd_q, one, one, ints(0, 1), ints(0, 1)), k[:1].expand(1, 2, 64))


@pytest.mark.parametrize("far", [1 << 23, 1 << 27, (1 << 27) + 8], ids=["2^23", "2^27", "past 2^27"])
@pytest.mark.parametrize("T,n", [(2, 40), (20, 72), (70, 2048)], ids=str)
def test_linear_rows_far_apart(engine, far, T, n):
    """The last position of each of several sequences: [:, -1] of [T, 2048, 4096] lies 2^23 elements apart."""
    store = torch.empty(T * far, dtype=torch.bfloat16, device="cuda")
    x, w = randn((T, 136), 0, torch.bfloat16).cuda(), randn((n, 136), 1, torch.bfloat16).cuda()
    r = randn((T, n), 2, torch.bfloat16).cuda()
    view = store.view(T, far)[:, -136:] if far % 136 else store.view(T, far)[:, :136]
    view.copy_(x)
    res = store.view(T, far)[:, :n]
    res.copy_(r)
    announce(f"linear T={T} n={n}, rows {view.stride(0)} apart")
    want = engine.linear(x, w, residual=r)
    assert torch.equal(engine.linear(view, w, residual=res), want)
    assert torch.equal(engine.linear(view, w, residual=res, out=res), want) and torch.equal(view, x)
    if n < 100 and T * far < 1 << 29:  # weight rows as far
        far_w = torch.empty(n * far, dtype=torch.bfloat16, device="cuda").view(n, far)[:, :136]
        far_w.copy_(w)
        assert torch.equal(engine.linear(view, far_w, residual=r), want)


def test_linear_strides_of_one_row_do_not_matter(engine):
    x, w = randn((1, 64), 0, torch.bfloat16).cuda(), randn((1, 64), 1, torch.bfloat16).cuda()
    announce("linear, strides of single rows")
    want = engine.linear(x, w, residual=x[:, :1])
    far = [t.as_strided(t.shape, (s, 1)) for t, s in ((x, 1 << 40), (w, 3), (x[:, :1], 1 << 50))]
    assert torch.equal(engine.linear(*far[:2], residual=far[2]), want)


@pytest.mark.parametrize("shape", [(0,), (2, 3, 0), (2, 0, 0), (1, 1, 1, 0)], ids=str)
def test_linear_of_no_columns_in_any_shape(engine, shape):
    announce(f"linear of {shape}")
    x, w = torch.zeros(shape, dtype=torch.float16, device="cuda"), torch.zeros(12, 0, dtype=torch.float16, device="cuda")
    b = randn((12,), 0, torch.float16).cuda()
    assert torch.equal(engine.linear(x, w, bias=b), b.expand(*shape[:-1], 12))
