"""GPU: paged_attention against its 64-bit definition (oracle/cache_ops.py), at
the lengths, pages, windows and layouts where it can go wrong.

Tolerances are packed_attention's (tests/test_gpu_model_ops.py): the same sums
in the same precision.  8-bit rows are compared with the values they stand for,
which the queries' type holds exactly.
"""
import math
from types import SimpleNamespace

import pytest
import torch

from adapterslotsplusplus_amd import WarpPipeEngine
from oracle import cache_ops as co
from tests.helpers import announce, gen, randn
from tests.test_gpu_model_ops import attention_tol, check

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def engine():
    return WarpPipeEngine()


def int32(v):
    return torch.tensor(v, dtype=torch.int32)


class Case:
    """Requests with their cache on the device: pages in a shuffled order, NaN in
    every row that holds no key, table entries past a request's pages nonsense."""

    def __init__(self, lens_q, lens_k, heads, kv_heads, dim, dtype, page=16, small=False, layout="heads", seed=0, spare=3, columns=2):
        self.lens_q, self.lens_k, self.dtype, self.dim = list(lens_q), list(lens_k), dtype, dim
        counts = [-(-n // page) for n in lens_k]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=gen(seed)).tolist()
        width = max(counts + [0]) + columns
        table = torch.randint(-5, 2 ** 30, (len(lens_k), width), generator=gen(seed + 1), dtype=torch.int32)
        rows = []
        at = 0
        for b, n in enumerate(counts):
            mine = order[at:at + n]
            at += n
            table[b, :n] = int32(mine)
            rows += [mine[j // page] * page + j % page for j in range(lens_k[b])]
        self.rows = torch.tensor(rows, dtype=torch.int64)
        self.table, self.page = table, page
        self.q = randn((sum(lens_q), heads, dim), seed + 2, dtype)
        self.scales = [None, None]
        self.dev, self.values = [], []
        for i in range(2):
            x = randn((len(rows), kv_heads, dim), seed + 3 + i, dtype)
            if small:
                v, e = co.quantise(x, torch.finfo(dtype).max)
                stored = torch.full((pages * page, kv_heads, dim), 0x7F, dtype=torch.uint8)
                stored[self.rows] = (v * torch.exp2(-e.double())[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
                codes = torch.full((pages * page, kv_heads), 255, dtype=torch.uint8)
                codes[self.rows] = (e + 127).to(torch.uint8)
                self.scales[i] = self.lay(codes.view(pages, page, kv_heads), layout)
                self.dev.append(self.lay(stored.view(pages, page, kv_heads, dim), layout).view(torch.float8_e4m3fn))
                x = v
            else:
                stored = torch.full((pages * page, kv_heads, dim), math.nan, dtype=dtype)
                stored[self.rows] = x
                self.dev.append(self.lay(stored.view(pages, page, kv_heads, dim), layout))
            full = torch.zeros(pages * page, kv_heads, dim, dtype=torch.float64)
            full[self.rows] = x.double()
            self.values.append(full.view(pages, page, kv_heads, dim))
        self.cu = int32([0] + self.lens_q).cumsum(0).int().cuda()
        self.kv = int32(self.lens_k).cuda()

    @staticmethod
    def lay(t, layout):
        t = t.cuda()
        if layout == "tokens":
            return t
        if layout == "heads":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        # Pages of one pool among others' rows.
        big = torch.zeros((t.size(0), 3, t.size(1), t.size(2)) + t.shape[3:], dtype=t.dtype, device="cuda")
        big[:, 1] = t
        return big[:, 1]

    def run(self, engine, q=None, **kw):
        return engine.paged_attention(self.q.cuda() if q is None else q, *self.dev, self.table.cuda(), self.cu, self.kv, k_scales=self.scales[0],
                                      v_scales=self.scales[1], return_lse=True, **kw)

    def want(self, scale=None, window=0, sinks=0):
        scale = self.dim ** -0.5 if scale is None else scale
        return co.paged_attention(self.q, *self.values, self.table, self.lens_q, self.lens_k, scale, window, sinks)

    def tolerance(self, out, lse, spread, reach):
        most = max(float(self.values[1].abs().max()), 0.0) if self.values[1].numel() else 0.0
        return attention_tol(out, lse, spread, reach, self.dim, self.lens_k + [0], most, self.dtype)


def attend(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, window=0, sinks=0, scale=None, **kw):
    announce(f"paged q={str(lens_q)[:60]} k={str(lens_k)[:60]} {heads}/{kv_heads}x{dim} {dtype} window={window}+{sinks} scale={scale} {kw}")
    c = Case(lens_q, lens_k, heads, kv_heads, dim, dtype, **kw)
    got, lse = c.run(engine, window=window, sinks=sinks, scale=scale)
    want = c.want(scale, window, sinks)
    tol, lse_tol = c.tolerance(*want)
    check(got, want[0], tol, "out")
    check(lse, want[1], lse_tol, "lse")
    return c, got, lse


FORMS = [(8, 2, 128, BF, dict()), (2, 2, 64, HF, dict(page=32, layout="tokens")), (7, 1, 96, HF, dict(small=True)),
         (32, 1, 64, BF, dict(small=True, page=64, layout="tokens")), (4, 4, 128, BF, dict(small=True, page=128, layout="pool")), (8, 1, 72, HF, dict(page=16, layout="pool"))]
FORM = pytest.mark.parametrize("heads,kv_heads,dim,dtype,kw", FORMS, ids=["8/2x128", "2/2x64", "7/1x96-8bit", "32/1x64-8bit", "4/4x128-8bit", "8/1x72"])

CACHED = [([1], [1]), ([1], [15]), ([1], [16]), ([1], [17]), ([1], [128]), ([1], [129]), ([1], [777]), ([1], [2049]), ([1, 1, 1, 1], [1, 64, 65, 500]),
          ([4, 2, 0, 5], [40, 700, 9, 5]), ([3, 8], [600, 33]), ([40], [300]), ([1, 0, 1], [0, 5, 3]), ([9], [4]), ([70, 1], [30, 0]), ([0, 0], [5, 3]),
          ([2] * 40, list(range(2, 202, 5)))]


@pytest.mark.parametrize("lens_q,lens_k", CACHED, ids=str)
@FORM
def test_cached(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, kw):
    """Few queries at the end of longer caches, more queries than keys (rows
    that see nothing), requests without queries or without keys."""
    attend(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, seed=len(lens_q), **kw)
    assert engine.device_errors() == 0


CHUNKS = [([33], [33]), ([64], [64]), ([65], [200]), ([127], [127]), ([128], [128]), ([129], [140]), ([256], [300]), ([300], [1000]), ([5, 0, 70, 1, 0, 130], [5, 9, 300, 40, 0, 131]),
          ([17, 1, 200], [1000, 1000, 1000]), ([100, 200, 3], [100, 150, 3])]


@pytest.mark.parametrize("lens_q,lens_k", CHUNKS, ids=str)
@FORM
def test_chunks(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, kw):
    attend(engine, lens_q, lens_k, heads, kv_heads, dim, dtype, seed=len(lens_q), **kw)
    assert engine.device_errors() == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (31, 4), (64, 64), (100, 130), (1000, 4), (2 ** 31 - 1, 2 ** 31 - 1), (5, 1000)])
@pytest.mark.parametrize("lens_q,lens_k", [([200], [200]), ([1, 1], [500, 3]), ([33, 5], [400, 64]), ([60], [900])], ids=str)
def test_window_and_first_keys(engine, lens_q, lens_k, window, sinks):
    attend(engine, lens_q, lens_k, 4, 2, 64, BF, window=window, sinks=sinks)
    attend(engine, lens_q, lens_k, 4, 1, 128, HF, window=window, sinks=sinks, small=True, page=32)


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 48, 56, 80, 96, 104, 112, 120])
def test_head_sizes(engine, dim, small):
    if small and dim % 16:
        pytest.skip("8-bit rows are multiples of 16 elements")
    attend(engine, [90, 3], [90, 3], 2, 1, dim, BF, seed=dim, small=small)
    attend(engine, [1, 2], [300, 70], 4, 2, dim, HF, seed=dim, small=small)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_page_sizes(engine, page):
    for layout in ("heads", "tokens", "pool"):
        attend(engine, [1, 3, 150], [page, 2 * page + 1, page + 140], 4, 2, 64, BF, page=page, layout=layout)
        attend(engine, [2], [3 * page - 1], 4, 2, 128, BF, page=page, layout=layout, small=True)


def test_more_requests_than_a_workgroup_has_threads(engine):
    lens_k = [b % 37 for b in range(700)]
    attend(engine, [1 if b % 5 else 0 for b in range(700)], lens_k, 2, 1, 64, BF)
    attend(engine, [1 if b != 300 else 90 for b in range(600)], [b % 11 + 1 if b != 300 else 333 for b in range(600)], 4, 1, 64, HF, small=True)


def test_long_caches(engine):
    """More granules of keys than are listed at a time, and many shares of a row."""
    attend(engine, [1], [20000], 2, 1, 64, BF)
    attend(engine, [2], [17001], 1, 1, 64, HF, small=True, page=256)
    attend(engine, [3, 1], [3, 16500], 32, 1, 64, BF, page=64)


def test_long_chunk_among_single_tokens(engine):
    n = 40
    lens_q, lens_k = [1 + b % 2 for b in range(n)], [3 * b + 2 for b in range(n)]
    lens_q[7], lens_k[7] = 200, 700
    for window, sinks in ((0, 0), (40, 3)):
        attend(engine, lens_q, lens_k, 8, 2, 128, BF, window=window, sinks=sinks)
        attend(engine, lens_q, lens_k, 1, 1, 64, BF, window=window, sinks=sinks, small=True)


def test_workgroups_of_several_requests(engine):
    """Shares that hold whole requests, ends of one and starts of the next."""
    lens_k = [(b * 97) % 1500 + 1 for b in range(150)]
    attend(engine, [1] * 150, lens_k, 8, 8, 64, BF)
    attend(engine, [b % 4 for b in range(150)], lens_k, 8, 4, 64, HF, page=32)


def device_want(c, window=0, sinks=0):
    """The definition in 64 bits on the device, for one request."""
    (n_q,), (n_k,) = c.lens_q, c.lens_k
    T, heads, dim = c.q.shape
    rows = c.rows.cuda()
    k, v = (t.reshape(-1, *t.shape[2:]).cuda()[rows] for t in c.values)
    group = heads // k.size(1)
    j, pos = torch.arange(n_k, device="cuda"), torch.arange(n_q, device="cuda")[:, None] + n_k - n_q
    hide = j > pos
    if window:
        hide |= (j <= pos - window) & (j >= sinks)
    out, spread = torch.zeros(T, heads, dim, dtype=torch.float64), torch.zeros(T, heads, dim, dtype=torch.float64)
    lse, reach = torch.zeros(T, heads, dtype=torch.float64), torch.zeros(T, heads, dtype=torch.float64)
    for h in range(heads):
        q, kk, vv = c.q[:, h].double().cuda(), k[:, h // group].double(), v[:, h // group].double()
        s = (q @ kk.t().contiguous() * dim ** -0.5).masked_fill(hide, -math.inf)
        p = torch.softmax(s, -1)
        out[:, h], spread[:, h], lse[:, h] = (p @ vv).cpu(), (p @ vv.abs()).cpu(), torch.logsumexp(s, -1).cpu()
        reach[:, h] = (q.abs() @ kk.abs().t().contiguous() * dim ** -0.5).masked_fill(hide, 0.0).amax(-1).cpu()
    return out, lse, spread, reach


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (5000, 300)])
def test_workgroups_that_walk_long_caches(engine, window, sinks, small):
    """As many row tiles as workgroups, each of more keys than are listed at a
    time; and single tokens, each of more than a wave's list."""
    for tokens, heads, kv_heads, dim, keys, dtype in ((700, 128, 64, 64, 9000, HF), (1500, 64, 16, 128, 11000, BF), (1, 1024, 1024, 16, 4500, BF)):
        announce(f"paged long walks {tokens} tokens {heads}/{kv_heads}x{dim} over {keys} {dtype} small={small} window={window}+{sinks}")
        c = Case([tokens], [keys], heads, kv_heads, dim, dtype, page=32, small=small)
        got, lse = c.run(engine, window=window, sinks=sinks)
        want = device_want(c, window, sinks)
        tol, lse_tol = c.tolerance(*want)
        check(got, want[0], tol, "out")
        check(lse, want[1], lse_tol, "lse")


def each_want(c):
    """device_want of each request."""
    parts, at_q, at_k = [], 0, 0
    for n_q, n_k in zip(c.lens_q, c.lens_k):
        parts.append(device_want(SimpleNamespace(lens_q=[n_q], lens_k=[n_k], q=c.q[at_q:at_q + n_q], rows=c.rows[at_k:at_k + n_k], values=c.values)))
        at_q, at_k = at_q + n_q, at_k + n_k
    return [torch.cat(t) for t in zip(*parts)]


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(128, 16, 64, BF), (32, 4, 128, HF), (64, 32, 32, BF)], ids=str)
def test_chunks_of_different_caches(engine, heads, kv_heads, dim, dtype, small):
    """More row tiles than workgroups over caches of different lengths, some longer
    than a workgroup's share, one twice as long; a single token among them."""
    more = 128 // heads  # as many rows of heads in all
    lens_q, lens_k = [120 * more, 1, 200 * more, 0, 140 * more, 60 * more], [6000, 700, 3100, 50, 2000, 16000]
    announce(f"paged chunks of different caches {heads}/{kv_heads}x{dim} {dtype} small={small}")
    c = Case(lens_q, lens_k, heads, kv_heads, dim, dtype, page=32, small=small)
    got, lse = c.run(engine)
    want = each_want(c)
    tol, lse_tol = c.tolerance(*want)
    check(got, want[0], tol, "out")
    check(lse, want[1], lse_tol, "lse")
    again = c.run(engine)
    assert torch.equal(got, again[0]) and torch.equal(lse, again[1])
    assert engine.device_errors() == 0


@pytest.mark.parametrize("lens_q,lens_k,heads", [([900, 450, 600, 500, 800], [900, 700, 600, 1600, 800], 64), ([450, 451] * 35, [450, 480] * 35, 8),
                                                 ([700] * 5, [700, 700, 700, 700, 30000], 64)], ids=["five", "seventy", "one-long"])
def test_many_row_tiles(engine, lens_q, lens_k, heads):
    """Several row tiles for each workgroup, of alike lengths and with one cache far longer."""
    announce(f"paged many row tiles, {len(lens_q)} requests")
    c = Case(lens_q, lens_k, heads, heads, 16, HF, page=64)
    got, lse = c.run(engine)
    want = each_want(c)
    tol, lse_tol = c.tolerance(*want)
    check(got, want[0], tol, "out")
    check(lse, want[1], lse_tol, "lse")
    again = c.run(engine)
    assert torch.equal(got, again[0]) and torch.equal(lse, again[1])


def test_scales(engine):
    for scale in (0.0, 1.0, 4.0, -0.3):
        attend(engine, [100], [300], 2, 2, 64, BF, scale=scale)
        attend(engine, [2], [900], 4, 1, 128, HF, scale=scale, small=True)


def test_views_and_outputs(engine):
    c = Case([60, 1, 9], [90, 130, 9], 6, 2, 40, BF)
    want, lse = c.run(engine)
    n = c.q.size(0)
    buf = torch.full((n, 10, 48), math.nan, dtype=BF, device="cuda")
    buf[:, :6, :40] = c.q.cuda()
    got, got_lse = c.run(engine, q=buf[:, :6, :40])
    assert torch.equal(got, want) and torch.equal(got_lse, lse)
    out = torch.full((n, 10, 48), math.nan, dtype=BF, device="cuda")
    got, _ = c.run(engine, out=out[:, 2:8, 8:])
    assert got.data_ptr() == out[:, 2:8, 8:].data_ptr() and torch.equal(got, want)
    assert int(torch.isnan(out).sum()) == out.numel() - got.numel()
    assert torch.equal(engine.paged_attention(c.q.cuda(), *c.dev, c.table.cuda(), c.cu, c.kv), want)
    wide = torch.zeros(3, c.table.size(1) + 5, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + c.table.size(1)] = c.table.cuda()
    assert torch.equal(engine.paged_attention(c.q.cuda(), *c.dev, wide[:, 2:2 + c.table.size(1)], c.cu, c.kv), want)


def test_rows_of_no_request_are_cleared(engine):
    for single in (True, False):
        c = Case([1, 1] if single else [70, 3], [20, 30] if single else [80, 30], 4, 2, 64, HF)
        want, lse = c.run(engine)
        n = c.q.size(0)
        q = torch.cat([torch.full((2, 4, 64), math.nan, dtype=HF), c.q, torch.full((5, 4, 64), math.nan, dtype=HF)]).cuda()
        out = torch.full_like(q, 3.0)
        c.cu = c.cu + 2
        got, got_lse = c.run(engine, q=q, out=out)
        assert torch.equal(got[2:2 + n], want) and torch.equal(got_lse[2:2 + n], lse)
        for rest in (slice(0, 2), slice(2 + n, None)):
            assert (got[rest] == 0).all() and (got_lse[rest] == -math.inf).all()
    none = engine.paged_attention(q, *c.dev, c.table[:0].cuda(), int32([0]).cuda(), int32([]).cuda())
    assert (none == 0).all()
    empty = engine.paged_attention(q[:0], *c.dev, c.table.cuda(), int32([0, 0, 0]).cuda(), c.kv)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
def test_pages_outside_the_cache_count_as_zeros(engine, small):
    for lens_q, lens_k in (([1, 2], [300, 50]), ([100, 1], [120, 70])):
        c = Case(lens_q, lens_k, 4, 2, 64, BF, small=small)
        engine.device_errors()
        c.run(engine)
        assert engine.device_errors() == 0
        good = c.table.clone()
        for bad in (-1, c.dev[0].size(0), 2 ** 31 - 1, -2 ** 31):
            c.table = good.clone()
            c.table[0, 1] = bad
            got, lse = c.run(engine)
            assert engine.device_errors() == 1
            # In the definition: a page of zeros.
            kept = c.values
            c.values = [torch.cat([v, torch.zeros(1, *v.shape[1:], dtype=v.dtype)]) for v in kept]
            c.table[0, 1] = kept[0].size(0)
            want = c.want()
            tol, lse_tol = c.tolerance(*want)
            c.values = kept
            check(got, want[0], tol, "out")
            check(lse, want[1], lse_tol, "lse")


def test_lengths_past_the_table_are_cut(engine):
    c = Case([2, 1], [64, 40], 4, 2, 64, BF, columns=0)
    c.kv = int32([1000, 40]).cuda()
    got, _ = c.run(engine)
    want = c.want()
    check(got, want[0], c.tolerance(*want)[0], "out")
    c.kv = int32([-5, 40]).cuda()
    got, lse = c.run(engine)
    assert (got[:2] == 0).all() and (lse[:2] == -math.inf).all()
    check(got[2:], want[0][2:], c.tolerance(*want)[0][2:], "out")


@pytest.mark.parametrize("small", [False, True], ids=["same", "8bit"])
def test_requests_that_share_pages(engine, small):
    """A prefix kept once: several rows of the table name the same pages, and a
    request may name one twice."""
    c = Case([1, 40, 3], [300, 300, 300], 8, 2, 128, BF, page=32, small=small)
    t = c.table.clone()
    t[1], t[2] = t[0], t[0]
    t[2, 4] = t[2, 3]
    got = engine.paged_attention(c.q.cuda(), *c.dev, t.cuda(), c.cu, c.kv, *c.scales)
    want = co.paged_attention(c.q, *c.values, t, c.lens_q, c.lens_k, 128 ** -0.5)
    check(got, want[0], c.tolerance(*want)[0], "out")


def test_unseen_keys_do_not_matter(engine):
    """NaN and infinity in keys and values that a query does not see leave it as it is."""
    for heads, kv_heads, small in ((2, 2, False), (8, 1, False), (8, 1, True)):
        for lens_q, lens_k in (([100, 2, 150], [100, 300, 150]), ([1, 3], [400, 90])):
            c = Case(lens_q, lens_k, heads, kv_heads, 64, BF, small=small)
            for window, sinks in ((0, 0), (40, 3)):
                clean, _ = c.run(engine, window=window, sinks=sinks)
                saved = [t.clone() for t in c.dev]
                # The last key of the first request is its last query's alone; with a window some keys before are seen by none of the others.
                row = int(c.rows[lens_k[0] - 1])
                for i, t in enumerate(c.dev):
                    (t.view(torch.uint8) if small else t)[row // c.page, row % c.page, :, 7 * i] = 0x7F if small else (math.nan, math.inf)[i]
                got, lse = c.run(engine, window=window, sinks=sinks)
                mine = lens_q[0] - 1
                assert torch.isnan(got[mine]).any()
                keep = torch.ones(len(got), dtype=torch.bool)
                keep[mine] = False
                assert torch.equal(got[keep], clean[keep]), (lens_q, window)
                c.dev = saved


def test_infinite_values_reach_who_sees_them(engine):
    c = Case([130, 2], [140, 300], 2, 1, 64, HF)
    row = int(c.rows[60])
    c.dev[1][row // 16, row % 16, 0, 5] = math.inf
    c.values[1][row // 16, row % 16, 0, 5] = math.inf
    got, _ = c.run(engine)
    want = c.want()
    seen = want[0].isinf()
    assert torch.equal(got.isinf().cpu(), seen) and seen[:, :, 5].any() and not seen[:, :, 6].any()
    ok = want[0].isfinite()
    tol = c.tolerance(want[0].nan_to_num(0, 0, 0), want[1], want[2].nan_to_num(0, 0, 0), want[3])[0]
    assert ((got.double().cpu() - want[0]).abs()[ok] <= tol.nan_to_num(1, 1, 1)[ok]).all()


def test_repeats_bit_for_bit(engine):
    for case in (Case([1] * 9, [3000, 1, 40, 700, 2000, 5, 5, 900, 1200], 8, 2, 128, BF), Case([300, 1], [2000, 900], 8, 2, 64, HF, small=True)):
        first = case.run(engine)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(case.run(engine), first))


def test_as_packed_attention_over_the_same_rows(engine):
    c = Case([300, 1, 20], [900, 2000, 20], 8, 2, 128, BF)
    out, lse = c.run(engine)
    k, v = (engine.read_cache(*c.dev, c.rows.cuda()))
    packed, plse = engine.packed_attention(c.q.cuda(), k, v, c.cu, int32([0] + c.lens_k).cumsum(0).int().cuda(), return_lse=True)
    want = c.want()
    tol, lse_tol = c.tolerance(*want)
    assert ((out.double() - packed.double()).abs().cpu() <= 2 * tol).all() and ((lse.double() - plse.double()).abs().cpu() <= 2 * lse_tol).all()


def test_caches_past_32_bits(engine):
    """Pages more than 2^32 bytes apart, and a stride between pages past 31 bits."""
    pages, size, heads, dim = 150000, 16, 8, 128  # 4.9 GB of keys
    k, v = (torch.empty(pages, heads, size, dim, dtype=BF, device="cuda").transpose(1, 2) for _ in range(2))
    c = Case([1, 40], [200, 70], 16, 8, 128, BF)
    far = [0, 1, pages // 2, pages - 1, pages - 2] + list(range(pages - 40, pages - 3))
    table = c.table.clone()
    at = 0
    for b, n in enumerate(c.lens_k):
        for j in range(-(-n // size)):
            k[far[at]], v[far[at]] = c.dev[0][table[b, j]], c.dev[1][table[b, j]]
            table[b, j] = far[at]
            at += 1
    got = engine.paged_attention(c.q.cuda(), k, v, table.cuda(), c.cu, c.kv)
    assert torch.equal(got, c.run(engine)[0])
    rows = torch.tensor([far[j // 16] * 16 + j % 16 for j in range(200)]).cuda()
    kk, vv = engine.read_cache(k, v, rows)
    old = engine.read_cache(*c.dev, c.rows[:200].cuda())
    assert torch.equal(kk, old[0]) and torch.equal(vv, old[1])
    engine.write_cache(vv, kk, k, v, rows)
    assert torch.equal(k[far[3], 5], vv[3 * 16 + 5])


def test_captured_and_replayed_with_other_lengths(engine):
    """One graph for any lengths that the table holds; two graphs share the scratch."""
    heads, kv, dim, page, n = 8, 2, 64, 16, 6
    cases = [Case([1] * n, [(7 * b + s * 131) % 900 + 1 for b in range(n)], heads, kv, dim, BF, seed=s) for s in range(3)]
    width, pages = max(c.table.size(1) for c in cases), max(c.dev[0].size(0) for c in cases)
    k, v = (torch.zeros(pages, page, kv, dim, dtype=BF, device="cuda") for _ in range(2))
    q, table = torch.zeros(n, heads, dim, dtype=BF, device="cuda"), torch.zeros(n, width, dtype=torch.int32, device="cuda")
    cu, lens = cases[0].cu.clone(), torch.ones(n, dtype=torch.int32, device="cuda")
    step = lambda **kw: engine.paged_attention(q, k, v, table, cu, lens, **kw)  # noqa: E731
    step()
    graphs = []
    for kw in (dict(), dict(window=100, sinks=4)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(**kw)
        graphs.append((g, out, kw))
    for _ in range(2):
        for c in cases:
            k[:c.dev[0].size(0)], v[:c.dev[1].size(0)] = c.dev[0], c.dev[1]
            q.copy_(c.q)
            table[:, :c.table.size(1)] = c.table.cuda()
            lens.copy_(c.kv)
            for g, out, kw in graphs:
                g.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, c.run(engine, **kw)[0])


def test_on_another_stream(engine):
    c = Case([1, 50], [300, 70], 4, 2, 64, BF)
    want = c.run(engine)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run(engine)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(engine):
    c = Case([1, 2], [30, 40], 4, 2, 64, BF)
    q, (k, v), t, cu, n = c.q.cuda(), c.dev, c.table.cuda(), c.cu, c.kv
    a = engine.paged_attention
    big = torch.zeros(2, 16, 2, 136, dtype=BF, device="cuda")
    for bad, kw in ((lambda: a(q.float(), k, v, t, cu, n), "fp16 or bf16"), (lambda: a(q.half(), k, v, t, cu, n), "pages must be"),
                    (lambda: a(q[:, :3], k, v, t, cu, n), "evenly"), (lambda: a(q[..., :32], k, v, t, cu, n), "heads, 64"),
                    (lambda: a(q, k, v, t.long(), cu, n), "int32"), (lambda: a(q, k, v, t, cu.long(), n), "int32"),
                    (lambda: a(q, k, v, t, cu[:2], n), "cu_seqlens_q"), (lambda: a(q, k, v, t[:1], cu, n), "block_table"),
                    (lambda: a(q, k, v, t.t().contiguous().t(), cu, n), "unit column"), (lambda: a(q, k, v, t, cu, n, window=-1), "window"),
                    (lambda: a(q, k, v, t, cu, n, sinks=4), "first keys"), (lambda: a(q, k, v, t, cu, n, window=4, sinks=-1), "window"),
                    (lambda: a(q, k, v, t.cpu(), cu, n), "CUDA"), (lambda: a(q, k, v, t, cu, n, out=q[:, :2]), "out must be"),
                    (lambda: a(q, k, v, t, cu, n, out=q[:1].expand(3, 4, 64)), "overlap"),
                    (lambda: a(torch.zeros(3, 4, 136, dtype=BF, device="cuda"), big, big, t, cu, n), "head size 136"),
                    (lambda: a(q, k[:, :8], v[:, :8], t, cu, n), "pages of 8")):
        with pytest.raises(RuntimeError, match=kw):
            bad()
