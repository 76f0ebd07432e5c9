"""The scan of microscaled 4-bit rows over rows that lie in patterns: pages dealt out in turn, runs of neighbours, and the orders that its lists
cannot hold.  References and the absence of a tolerance: as in test_gpu_mx4_lengths.py.

A query whose lists overflow is marked in the workspace and done over by one workgroup, which is right but slow (milliseconds at a million
rows); which queries were marked is read from the workspace, so that a pattern that ought to be ordinary is not merely answered right."""
import numpy as np
import pytest

from test_gpu_mx4_lengths import check, engines, random_bits, unit_rows, want_scan  # noqa: F401 (engines is a fixture)

pytestmark = pytest.mark.gpu


def scan_marked(mx, q, r, k, words=None):
    """-> ((ids, values, counts), which queries were done over); at most 8192 queries, more than 8"""
    import torch
    nq, n = q.shape[0], r.shape[0]
    h = mx._engine()
    need = mx.L.mvdb_mx4_scan_workspace(h, nq, n, k)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    ids, val, cnt = (torch.empty(s, dtype=t, device="cuda") for s, t in
                     (((nq, k), torch.int32), ((nq, k), torch.float32), ((nq,), torch.int32)))
    ok = mx.L.mvdb_mx4_scan_many_dev(h, q.data_ptr(), nq, r.data_ptr(), n, k, None if words is None else words.data_ptr(), ids.data_ptr(),
                                     val.data_ptr(), cnt.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert ok == 1
    up = lambda b: (b + 255) // 256 * 256
    at = up(nq * 128 * 8) + up(nq * 8) + up(nq * 4)  # best keys, bounds, numbers of best keys
    return (ids, val, cnt), ws[at : at + 4 * nq].view(torch.int32) != 0


def words_of(keep):
    import torch
    bits = torch.nn.functional.pad(keep, (0, -keep.numel() % 32)).view(-1, 32)
    return (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)


@pytest.mark.parametrize("nq", [40, 300])
@pytest.mark.parametrize("period", [2, 3, 4, 5, 6, 7, 8, 12, 16])
def test_pages_in_turn_filtered(engines, nq, period):
    """Pages of 64 rows dealt out in turn, the filter keeps those of one owner."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(period)
    n, mx = 500003, engines(64)
    q, r = mx.quantize(unit_rows(g, nq, 64)), mx.quantize(unit_rows(g, n, 64))
    for owner in (1, period - 1):
        keep = (torch.arange(n, device="cuda") // 64) % period == owner
        got, marked = scan_marked(mx, q, r, 10, words_of(keep))
        check(got, want_scan(mx, q, r, 10, keep))
        assert not marked.any()


@pytest.mark.parametrize("nq", [40, 300])
@pytest.mark.parametrize("period", [2, 5, 7, 8, 16])
def test_pages_in_turn_better(engines, nq, period):
    """No filter, but one page in `period` holds rows that every query likes better than all others."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(period)
    n, mx = 500003, engines(64)
    x = unit_rows(g, n, 64)
    x[:, 0] = torch.where((torch.arange(n, device="cuda") // 64) % period == period - 1, 1.0, -1.0)
    y = unit_rows(g, nq, 64)
    y[:, 0] = 2
    q, r = mx.quantize(y), mx.quantize(x)
    got, marked = scan_marked(mx, q, r, 10)
    check(got, want_scan(mx, q, r, 10))
    assert not marked.any()


@pytest.mark.parametrize("nq", [40, 300])
def test_runs_of_neighbours(engines, nq):
    """Each query has a run of 20 pages of rows that it likes better than all others, somewhere."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(nq)
    n, mx = 500003, engines(64)
    x, y = unit_rows(g, n, 64), unit_rows(g, nq, 64)
    for i in range(nq):
        at = int(torch.randint(0, n - 1280, (1,), generator=g, device="cuda"))
        x[at : at + 1280] = 0.7 * y[i] + 0.3 * x[at : at + 1280]
    q, r = mx.quantize(y), mx.quantize(x)
    got, marked = scan_marked(mx, q, r, 10)
    check(got, want_scan(mx, q, r, 10))
    assert not marked.any()


def tile_order(tiles):
    """The order in which a scan takes its tiles of 64 rows: (p M) mod tiles, M the first near tiles / golden ratio whose continued
    fraction with tiles has no term above 5."""
    start, best = int(0.6180339887498949 * tiles), (1 << 32, 1)
    for i in range(64):
        m = start - (i + 1) // 2 if i & 1 else start + i // 2
        if not 0 < m < tiles or best[0] <= 5:
            continue
        a, b, term = tiles, m, 0
        while b:
            term = max(term, a // b)
            a, b = b, a % b
        if a == 1 and term < best[0]:
            best = (term, m)
    return np.arange(tiles, dtype=np.int64) * best[1] % tiles


@pytest.mark.parametrize("share", [1.0, 0.4])
@pytest.mark.parametrize("nq,k", [(12, 10), (300, 10), (300, 100), (2200, 10), (2200, 100)])
@pytest.mark.parametrize("dim", [64, 100, 384, 512, 768, 1000])
def test_orders_that_overflow(engines, dim, nq, k, share):
    """The first tiles that a scan takes hold poor rows and all others good ones: every good row beats the bound, more than any list holds."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(dim + nq)
    mx, tiles = engines(dim), 1500
    n = 64 * tiles - 37
    q = mx.quantize(1 + 0.5 * torch.randint(0, 2, (nq, dim), generator=g, device="cuda"))
    order = torch.from_numpy(tile_order(tiles)).cuda()
    words, keep = random_bits(g, n, share) if share < 1 else (None, None)
    some = False
    for first in (32, 215):  # level 0 alone, and with the level that follows it
        good = torch.ones(tiles, dtype=torch.bool, device="cuda")
        good[order[:first]] = False
        x = 1 + 0.5 * torch.randint(0, 2, (n, dim), generator=g, device="cuda")
        x *= torch.where(good[torch.arange(n, device="cuda") // 64], 1.0, -1.0)[:, None]
        r = mx.quantize(x)
        got, marked = scan_marked(mx, q, r, k, words)
        check(got, want_scan(mx, q, r, k, keep))
        some |= bool(marked.any())
    assert some


@pytest.mark.parametrize("share", [1.0, 0.3])
def test_some_queries_overflow(engines, share):
    """Queries that are done over beside queries that are not, a wave a selection: what the others found stays."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    mx, tiles, nq, k = engines(128), 1500, 2200, 10
    n = 64 * tiles
    order = torch.from_numpy(tile_order(tiles)).cuda()
    good = torch.ones(tiles, dtype=torch.bool, device="cuda")
    good[order[:32]] = False
    x = unit_rows(g, n, 128)
    x[:, :64] = 0.25 * torch.where(good[torch.arange(n, device="cuda") // 64], 1.0, -1.0)[:, None]
    y = unit_rows(g, nq, 128)
    y[:, :64] = torch.where(torch.arange(nq, device="cuda") % 3 == 0, 1.0, 0.0)[:, None]  # every third query likes the late rows
    q, r = mx.quantize(y), mx.quantize(x)
    words, keep = random_bits(g, n, share) if share < 1 else (None, None)
    got, marked = scan_marked(mx, q, r, k, words)
    check(got, want_scan(mx, q, r, k, keep))
    assert marked[::3].all() and not marked[1::3].any() and not marked[2::3].any()


@pytest.mark.parametrize("page", [32, 128, 3000, 20000])
@pytest.mark.parametrize("nq,dim", [(12, 384), (300, 64), (300, 1000), (2200, 64)])
def test_overflow_with_gaps(engines, nq, dim, page):
    """Queries that are done over where the filter leaves out whole groups of rows, the store ending inside one of either kind."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(page)
    mx, tiles, some = engines(dim), 1500, False
    q = mx.quantize(1 + 0.5 * torch.randint(0, 2, (nq, dim), generator=g, device="cuda"))
    order = torch.from_numpy(tile_order(tiles)).cuda()
    good = torch.ones(tiles, dtype=torch.bool, device="cuda")
    good[order[:215]] = False
    for n, odd in ((64 * tiles, 0), (64 * tiles - 63, 1), (64 * tiles - 1, 0)):
        at = torch.arange(n, device="cuda")
        x = 1 + 0.5 * torch.randint(0, 2, (n, dim), generator=g, device="cuda")
        x *= torch.where(good[at // 64], 1.0, -1.0)[:, None]
        r = mx.quantize(x)
        keep = (at // page) % 2 == odd
        got, marked = scan_marked(mx, q, r, 10, words_of(keep))
        check(got, want_scan(mx, q, r, 10, keep))
        some |= bool(marked.any())
    assert some
