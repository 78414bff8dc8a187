"""GPU: the memory that the operators around the apply keep."""
import gc

import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from tests.helpers import announce, randn

pytestmark = pytest.mark.gpu

SCRATCH = 256 << 20


def free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def test_scratch_belongs_to_engines_that_use_it():
    announce("operators' scratch: engines with and without calls")
    x, w = randn((2, 64), 0, torch.bfloat16).cuda(), randn((16, 64), 1, torch.bfloat16).cuda()
    WarpPipeEngine().linear(x, w)  # whatever a process allocates once
    gc.collect()
    at = free()
    engines = [WarpPipeEngine() for _ in range(3)]
    for e in engines:
        assert e.build_seg_bounds(torch.zeros(4, dtype=torch.int64, device="cuda"))
    idle = at - free()
    assert idle < SCRATCH, f"three engines that run no operator hold {idle >> 20} MiB"
    for e in engines[:2]:
        e.linear(x, w)
        e.linear(x, w)
    # (Device memory is counted in pages of 2 MiB, and not these calls' alone.)
    assert round((at - free() - idle) / SCRATCH) == 2
    del engines, e
    gc.collect()
    assert at - free() < SCRATCH


def test_first_call_captured():
    """The scratch of an engine whose first call is recorded into a graph."""
    announce("operators: first call in a capture")
    x, w = randn((2, 16384), 0, torch.bfloat16).cuda(), randn((80, 16384), 1, torch.bfloat16).cuda()
    want = WarpPipeEngine().linear(x, w)
    engine = WarpPipeEngine()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = engine.linear(x, w)
    for seed in range(3):
        x.copy_(randn((2, 16384), seed, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, engine.linear(x, w)), f"replay {seed}"
        if seed == 0:
            assert torch.equal(got, want)
