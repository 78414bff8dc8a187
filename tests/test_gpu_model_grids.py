"""GPU: calls of the model operators that would take a grid of 2^32 threads or
more run in several launches, or are refused."""
import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from tests.helpers import announce

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


@pytest.mark.parametrize("top", [0, 2])
def test_logprobs_of_many_rows(engine, top):
    rows, vocab = (1 << 23) + 1001, 8
    announce(f"logprobs of {rows} rows, top {top}")
    logits = torch.empty(rows, vocab, dtype=BF, device="cuda").normal_()
    ids = torch.randint(-1, vocab, (rows,), dtype=torch.int32, device="cuda")
    got = engine.token_logprobs(logits, ids, top)
    for a in range(0, rows, 1 << 21):
        part = slice(a, min(rows, a + (1 << 21)))
        for all_rows, some in zip(got, engine.token_logprobs(logits[part], ids[part], top)):
            assert torch.equal(all_rows[part], some)
    assert engine.device_errors() == 0


def test_linear_refuses_what_no_grid_holds(engine):
    """2^30 tokens, all of one row, by one output: 2^24 tiles of 64 tokens, 256 threads each."""
    T = 1 << 30
    announce(f"linear of {T} tokens")
    x, w = torch.ones(1, 8, dtype=BF, device="cuda").expand(T, 8), torch.ones(1, 8, dtype=BF, device="cuda")
    out = torch.zeros(T, 1, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="too many for one call"):
        engine.linear(x, w, out=out)
    n = T - (1 << 20)
    engine.linear(x[:n], w, out=out[:n])
    assert (out[:n] == 8).all() and (out[n:] == 0).all()


def test_packed_attention_refuses_what_no_grid_holds(engine):
    """2^24 single tokens, a workgroup of 256 threads each."""
    n = 1 << 24
    announce(f"packed attention of {n} sequences")
    q = torch.zeros(1, 1, 8, dtype=BF, device="cuda").expand(n, 1, 8)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="too many for one call"):
        engine.packed_attention(q, q, q, cu)
