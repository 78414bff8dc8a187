"""GPU: packed_attention at the ends of its ranges: bounds that fall (the calls
after such a one answer as on a new engine), windows past 31 bits."""
import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from tests.helpers import announce, randn

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


# bounds that fall, and bounds that rise of as many sequences whose keys are split the same way
KEY_CHUNKS = ([0, 1, 2, 3, 4, 5], [0, 8000, 0, 8000, 0, 8000], [0, 1, 2, 3, 4, 5], [0, 1600, 3200, 4800, 6400, 8000])
ROW_TILES = ([0, 300, 0, 300], [0, 8000, 0, 8000], [0, 140, 150, 300], [0, 3900, 4000, 8000])


@pytest.mark.parametrize("cu_q,cu_k,next_q,next_k", [KEY_CHUNKS, ROW_TILES], ids=["key chunks", "row tiles"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (2, 2, 128)], ids=str)
def test_falling_bounds_leave_the_counters_at_zero(cu_q, cu_k, next_q, next_k, heads, kv_heads, dim):
    announce(f"attention, falling bounds q={cu_q} k={cu_k} heads={heads}/{kv_heads}x{dim}")
    T, S = max(cu_q), max(cu_k)
    q = randn((T, heads, dim), 0, torch.bfloat16).cuda()
    k, v = (randn((S, kv_heads, dim), i, torch.bfloat16).cuda() for i in (1, 2))
    x, w = randn((2, 16384), 3, torch.bfloat16).cuda(), randn((80, 16384), 4, torch.bfloat16).cuda()
    logits, ids = randn((3, 60000), 5, torch.float32).cuda(), torch.tensor([1, 2, 3]).cuda()

    def valid(engine):
        out = [*engine.packed_attention(q, k, v, ints(next_q), ints(next_k), return_lse=True), engine.linear(x, w),
               *engine.token_logprobs(logits, ids, top=3)]
        return [t.clone() for t in out]

    want = valid(WarpPipeEngine())
    engine = WarpPipeEngine()
    for _ in range(3):
        engine.packed_attention(q, k, v, ints(cu_q), ints(cu_k))
        for got, t in zip(valid(engine), want):
            assert torch.equal(got, t)


@pytest.mark.parametrize("n_q,n_k", [(1000, 500), (5, 900), (300, 300)], ids=str)
def test_windows_wider_than_the_keys(n_q, n_k):
    """As no window, up to and past the largest 32-bit number."""
    engine = WarpPipeEngine()
    q, k = randn((n_q, 2, 64), 0, torch.bfloat16).cuda(), randn((n_k, 2, 64), 1, torch.bfloat16).cuda()
    cu_q, cu_k = ints([0, n_q]), ints([0, n_k])
    want = engine.packed_attention(q, k, k, cu_q, cu_k)
    for window in (n_k, 2 ** 31 - 1 - n_q, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 70):
        announce(f"attention q={n_q} k={n_k} window={window}")
        assert torch.equal(engine.packed_attention(q, k, k, cu_q, cu_k, window=window), want), window
    with pytest.raises(RuntimeError, match="window"):
        engine.packed_attention(q, k, k, cu_q, cu_k, window=-(2 ** 32))
