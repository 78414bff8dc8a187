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
