"""Host-side logic of the multi-tenant decoder (no GPU): where a packed cache's
kept and new rows go, and the checks of shapes."""
import pytest
import torch

from adapterslotsplusplus_amd.prompt_scoring import DecoderLayer, PackedCache, TenantDecoder


def test_cache_keeps_sequences_in_order():
    cache = PackedCache(layers=1, sequences=3)
    have = [torch.zeros(0), torch.zeros(0), torch.zeros(0)]
    at = 0.0
    for lens in ([2, 0, 3], [1, 4, 0], [0, 0, 0], [2, 1, 1]):
        rows = []
        for b, n in enumerate(lens):
            new = torch.arange(n) + at
            at += n
            rows.append(new)
            have[b] = torch.cat([have[b], new])
        cache.grow(lens, "cpu")
        flat = torch.cat(rows).view(-1, 1, 1)
        k, v = cache.add(0, flat, -flat)
        assert torch.equal(k.flatten(), torch.cat(have)) and torch.equal(v.flatten(), -torch.cat(have))
        assert cache.cu.tolist() == [0] + torch.tensor([len(h) for h in have]).cumsum(0).tolist()
        assert cache.lens == [len(h) for h in have]


def test_cache_refuses_another_batch():
    cache = PackedCache(layers=1, sequences=2)
    with pytest.raises(RuntimeError, match="1 sequences, the cache has 2"):
        cache.grow([3], "cpu")


@pytest.mark.parametrize("heads,kv_heads", [(4, 3), (0, 1), (5, 1)])
def test_heads_must_fit_the_projection(heads, kv_heads):
    z = torch.zeros(1)
    layer = DecoderLayer(z, torch.zeros(64, 32), z, z, z, z)
    with pytest.raises(RuntimeError, match="w_qkv"):
        TenantDecoder(None, z, [layer], z, z, heads, kv_heads)
