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
