"""Host-side: a paged cache's pages, slots and positions, and a decoder's steps
over one on an engine that computes on the CPU (no GPU)."""
import pytest
import torch

from adapterslotsplusplus_amd.prompt_scoring import DecoderLayer, PackedCache, PagedCache, TenantDecoder
from adapterslotsplusplus_amd.rotary import Rotary, frequencies
from oracle import cache_ops as co
from tests.test_prompt_scoring_steps_host import DIM, HEADS, KV, VOCAB, HostEngine, parts

SIZE = 16


class PagedHostEngine(HostEngine):
    """The plain operators over pages (rows of the pages' own type)."""

    def rotate_heads(self, q, k, positions, rotary, q_norm=None, k_norm=None, eps=1e-6, q_out=None, k_out=None):
        freq = frequencies(rotary.dim)[0] if rotary is not None else []
        for x, w, out in ((q, q_norm, q_out), (k, k_norm, k_out)):  # out may be x
            out.copy_(co.rotate(co.norm_heads(x, w, eps), positions, freq))

    def rotate_into_cache(self, q, k, v, positions, rotary, k_pages, v_pages, slots, k_scales=None, v_scales=None,
                          q_norm=None, k_norm=None, eps=1e-6, q_out=None):
        turned = k.clone()
        self.rotate_heads(q, k, positions, rotary, q_norm, k_norm, eps, q_out, turned)
        self.write_cache(turned, v, k_pages, v_pages, slots)

    def write_cache(self, k, v, k_pages, v_pages, slots, k_scales=None, v_scales=None):
        assert len(set(slots.tolist())) == len(slots)
        for rows, pages in ((k, k_pages), (v, v_pages)):
            pages.view(-1, *pages.shape[2:])[slots] = rows

    def paged_attention(self, q, k_pages, v_pages, block_table, cu_q, kv_lens, k_scales=None, v_scales=None):
        return co.paged_attention(q.double(), k_pages.double(), v_pages.double(), block_table, cu_q.diff().tolist(),
                                  kv_lens.tolist(), DIM ** -0.5)[0].float()


def decoder(engine, rotary=True, norms=True):
    g = torch.Generator().manual_seed(0)

    def w(*shape):
        return torch.randn(*shape, generator=g) * 0.3

    ls = [DecoderLayer(w(16), w((HEADS + 2 * KV) * DIM, 16), w(16, HEADS * DIM), w(16), w(40, 16), w(16, 20))
          for _ in range(2)]
    return TenantDecoder(engine, w(VOCAB, 16), ls, w(16), w(VOCAB, 16), HEADS, KV,
                         rotary=Rotary(DIM, device="cpu") if rotary else None,
                         head_norms=[(1 + w(DIM), None), (1 + w(DIM), 1 + w(DIM))] if norms else None)


def step(model, rows, cache=None):
    lens = [len(p) for p in rows]
    ids = torch.cat(rows)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    who = torch.full((len(ids),), -1)
    if cache is None:
        return model.score(ids, cu, who, lens)
    return model.verify(ids, cu, who, lens, cache)


def test_pages_hold_whole_sequences():
    cache = PagedCache(1, 3, pages=8, kv_heads=1, dim=8, dtype=torch.float32, page_size=SIZE)
    have = [[], [], []]
    store = {}
    at = 0
    for lens in ([17, 0, 3], [15, 30, 0], [0, 0, 0], [1, 2, 14]):
        cache.grow(lens, "cpu")
        new = list(range(at, at + sum(lens)))
        at += len(new)
        store.update(zip(cache.slots.tolist(), new))
        i = 0
        for b, n in enumerate(lens):
            assert cache.positions[i:i + n].tolist() == list(range(len(have[b]), len(have[b]) + n))
            have[b] += new[i:i + n]
            i += n
        for b in range(3):
            row = cache.table[b].tolist()
            assert [store[row[j // SIZE] * SIZE + j % SIZE] for j in range(len(have[b]))] == have[b]
        assert cache.lens == cache.kv_lens.tolist() == [len(h) for h in have]
        pages = [p for t in cache.tables for p in t] + cache.free
        assert sorted(pages) == list(range(8)) and [len(t) for t in cache.tables] == [-(-len(h) // SIZE) for h in have]


def test_cut_frees_whole_pages():
    cache = PagedCache(1, 2, pages=5, kv_heads=1, dim=8, dtype=torch.float32, page_size=SIZE)
    cache.grow([33, 32], "cpu")
    first = [list(t) for t in cache.tables]
    assert cache.free == []
    cache.cut([17, 32])
    assert cache.lens == [17, 32] and cache.tables == [first[0][:2], first[1]] and cache.free == first[0][2:]
    cache.cut([17, 0])
    assert cache.tables[1] == [] and len(cache.free) == 3
    cache.grow([0, 40], "cpu")
    assert cache.lens == [17, 40] and cache.free == []
    for bad in ([18, 0], [-1, 0], [17]):
        with pytest.raises(RuntimeError, match="cannot stay"):
            cache.cut(bad)


@pytest.mark.parametrize("lens,message", [([81, 0], "takes 6 pages, 5 are free"), ([1], "1 sequences, the cache has 2")])
def test_a_step_that_does_not_fit_is_refused(lens, message):
    cache = PagedCache(1, 2, pages=5, kv_heads=1, dim=8, dtype=torch.float32, page_size=SIZE)
    with pytest.raises(RuntimeError, match=message):
        cache.grow(lens, "cpu")
    assert cache.lens == [0, 0] and cache.free == [0, 1, 2, 3, 4] and cache.tables == [[], []]


@pytest.mark.parametrize("size", [0, 8, 24, -16])
def test_page_sizes(size):
    with pytest.raises(RuntimeError, match="power of two"):
        PagedCache(1, 1, pages=1, kv_heads=1, dim=8, dtype=torch.float32, page_size=size)


@pytest.mark.parametrize("rotary,norms", [(True, True), (True, False), (False, True), (False, False)])
def test_both_caches_say_the_same(rotary, norms):
    model = decoder(PagedHostEngine(), rotary, norms)
    packed, paged = None, model.paged_cache(3, pages=9, page_size=SIZE)
    for i, lens in enumerate(([20, 1, 0], [3, 15, 2], [0, 0, 0], [1, 1, 1])):
        rows = parts(i, *lens)
        want = step(model, rows, packed)
        want, packed = want if packed is None else (want, packed)
        got = step(model, rows, paged)
        assert torch.allclose(got.logprobs, want.logprobs, atol=1e-5) and paged.lens == packed.lens
        if sum(lens):
            assert torch.equal(packed.positions("cpu"), paged.positions)


def test_head_norms_are_for_every_layer():
    z = torch.zeros(1)
    layer = DecoderLayer(z, torch.zeros(64, 32), z, z, z, z)
    with pytest.raises(RuntimeError, match="head_norms for 1 of 2 layers"):
        TenantDecoder(None, z, [layer, layer], z, z, 2, 1, head_norms=[(None, None)])


def test_drafts_taken_back():
    """A cache cut after drafts goes on as one that never saw them."""
    model = decoder(PagedHostEngine())
    first, drafts, more = parts(1, 17, 4), parts(2, 20, 3), parts(3, 2, 14)
    caches = [model.paged_cache(2, pages=6, page_size=SIZE) for _ in range(2)]
    for cache in caches:
        step(model, first, cache)
    step(model, drafts, caches[0])
    caches[0].cut([17, 4])
    got, want = (step(model, more, cache) for cache in caches)
    assert torch.equal(got.logprobs, want.logprobs) and caches[0].lens == caches[1].lens


@pytest.mark.parametrize("refuse,message", [("tokens", "max_tokens"), ("top", "refused"), (None, "pages")])
def test_a_step_that_fails_gives_its_pages_back(refuse, message):
    engine = PagedHostEngine()
    model = decoder(engine)
    cache = model.paged_cache(2, pages=4, page_size=SIZE)
    step(model, parts(1, 17, 4), cache)
    other = model.paged_cache(2, pages=4, page_size=SIZE)
    step(model, parts(1, 17, 4), other)
    before = [list(t) for t in cache.tables], list(cache.free)
    engine.refuse = refuse
    with pytest.raises(RuntimeError, match=message):
        step(model, parts(2, 40, 1) if refuse is None else parts(2, 2, 15), cache)
    assert cache.lens == [17, 4] and (cache.tables, cache.free) == before
    engine.refuse = None
    more = parts(4, 3, 13)
    assert torch.equal(step(model, more, cache).logprobs, step(model, more, other).logprobs)


@pytest.mark.parametrize("kind", ["packed", "paged"])
def test_sequences_do_not_grow_by_fewer_than_no_tokens(kind):
    """A negative length is refused before anything of the cache changes (its pages
    would be handed out twice, or lost)."""
    model = decoder(PagedHostEngine())
    cache = model.paged_cache(2, pages=6, page_size=SIZE) if kind == "paged" else PackedCache(2, 2)
    other = model.paged_cache(2, pages=6, page_size=SIZE)
    for c in (cache, other):
        step(model, parts(1, 33, 4), c)
    ids = torch.cat(parts(2, 2))
    kept = cache.state()
    for lens in ([-1, 3], [3, -1]):
        with pytest.raises(RuntimeError, match="none by fewer than 0"):
            cache.grow(lens, "cpu")
        with pytest.raises(RuntimeError, match="none by fewer than 0"):
            model.verify(ids, torch.tensor([0, 2, 2], dtype=torch.int32), torch.tensor([-1, -1]), lens, cache)
    assert cache.lens == [33, 4]
    if kind == "paged":
        assert cache.state()[:3] == kept[:3] and sorted([p for t in cache.tables for p in t] + cache.free) == list(range(6))
    more = parts(3, 1, 14)
    assert torch.allclose(step(model, more, cache).logprobs, step(model, more, other).logprobs, atol=1e-5)
