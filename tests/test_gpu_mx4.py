"""Microscaled 4-bit rows on the GPU against the 64-bit oracle (oracle/mx4_oracle.py).

Tolerances.  Quantisation and expansion: none, every byte and value is determined.  Products: a product of two values is a
multiple of 1/4 of its two scales' product and at most 36 of it, so a sum over `dim` components whose scales span at most
2^w needs 2 + log2(36 dim) + w bits; up to 24 of them an f32 sum is exact in any order, and the test asks for equality.  Beyond
that a matrix instruction adds 64 products and the accumulator, each cut at 2^-24 of the largest of them at worst, so with P =
sum |q_i r_i| the error is at most 65 * 2^-24 * P for each of dim / 64 instructions."""
import ctypes as C

import numpy as np
import pytest

from oracle import mx4_oracle as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engines(gpu):
    import torch
    from minivectordb_amd import HipBridge
    from minivectordb_amd.pipeline import ResidentMx4
    made = {}

    def get(dim):
        if dim not in made:
            b = HipBridge(device=0)
            b.init(dict(dim=dim, m=8, ef=50, capacity=8, seed=1))
            made[dim] = ResidentMx4(b, torch.device("cuda", 0))
        return made[dim]

    yield get
    torch.cuda.synchronize()
    for mx in made.values():
        mx.b.close()


def _unit(rng, n, dim, centres=64):
    c = rng.standard_normal((centres, dim))
    x = c[rng.integers(0, centres, n)] + rng.standard_normal((n, dim))
    return (x / np.linalg.norm(x, axis=1, keepdims=True)).astype(np.float32)


def _to(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _specials(dim):
    x = np.zeros((12, dim), np.float32)
    tiny = np.float32(2.0**-149)
    grid = np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.99], np.float32)
    x[0] = np.resize(np.concatenate([grid, -grid]), dim)         # every tie and every magnitude, scale 1
    x[1] = -0.0
    x[2] = np.resize(np.array([1, np.nan, 2], np.float32), dim)
    x[3, 0] = np.inf                                             # only the first block is bad
    x[3, dim - 1] = 1
    x[4] = -np.inf
    x[5] = np.resize(np.array([tiny, -tiny, 3 * tiny], np.float32), dim)
    x[6] = np.resize(np.array([2.0**-126, 2.0**-127, -(2.0**-125), 2.0**-128], np.float32), dim)
    x[7] = np.finfo(np.float32).max
    x[8] = np.nextafter(np.float32(8), np.float32(0))
    x[9] = 8
    x[10] = np.resize(np.ldexp(np.float32(1), np.arange(-60, 60)).astype(np.float32), dim)
    x[11] = np.resize(np.array([0, 0, 0, 1e-30], np.float32), dim)
    return x


@pytest.mark.parametrize("dim", [4, 32, 60, 64, 100, 384, 512, 1000, 1024, 4096])
@pytest.mark.parametrize("rows", [1, 37, 259])
def test_quantise_f32(engines, dim, rows):
    rng = np.random.default_rng(dim * 1000 + rows)
    x = rng.standard_normal((rows, dim)).astype(np.float32) * np.exp2(rng.integers(-12, 12, (rows, 1))).astype(np.float32)
    x[: min(12, rows)] = _specials(dim)[: min(12, rows)]
    mx = engines(dim)
    got = mx.quantize(_to(x))
    want = M.pack(x)
    assert np.array_equal(got.cpu().numpy(), want)
    v = mx.expand(got).cpu().numpy()
    assert v.dtype == np.float32 and np.array_equal(v, M.values(want, dim).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,pad,first", [(100, 7, 0), (384, 24, 8), (1000, 1, 3), (64, 0, 0)])
def test_quantise_types_and_strides(engines, kind, dim, pad, first):
    import torch
    dt = dict(bf16=torch.bfloat16, f16=torch.float16, f32=torch.float32)[kind]
    rng = np.random.default_rng(dim + pad)
    wide = _to(rng.standard_normal((83, dim + pad + first)).astype(np.float32)).to(dt)
    wide[5, first + 2] = float("nan")
    wide[6, first + 3] = float("inf")
    wide[7, first:] *= 2.0**-16 if kind == "f16" else 2.0**-100  # f16: subnormal values
    x = wide[:, first : first + dim]
    assert np.array_equal(engines(dim).quantize(x).cpu().numpy(), M.pack(x.double().cpu().numpy()))
    # one row of a wider buffer, rows in another order of memory
    assert np.array_equal(engines(dim).quantize(x[40:41]).cpu().numpy(), M.pack(x[40:41].double().cpu().numpy()))
    assert np.array_equal(engines(dim).quantize(x[::3]).cpu().numpy(), M.pack(x[::3].double().cpu().numpy()))


def test_quantise_refuses(engines):
    import torch
    from minivectordb_amd import MvdbError
    mx = engines(64)
    x = torch.zeros((4, 128), device="cuda")
    for bad in (x, x[:, ::2], x[:, :64].double(), x[:, :64].to(torch.int8), x[0, :64], x[:1, :64].expand(4, 64)):
        with pytest.raises(MvdbError):
            mx.quantize(bad)
    p = torch.zeros((4, 48), dtype=torch.uint8, device="cuda")
    for bad in (p[:, :32], p.to(torch.int8), torch.zeros((4, 96), dtype=torch.uint8, device="cuda")[:, :48], p[0]):
        with pytest.raises(MvdbError):
            mx.expand(bad)
    with pytest.raises(MvdbError):
        mx.product(p, p, out=torch.zeros((4, 5), device="cuda"))
    with pytest.raises(MvdbError):
        mx.product(p, p, out=torch.zeros((4, 4), device="cuda", dtype=torch.bfloat16))
    with pytest.raises(MvdbError):
        mx.product(p, p, out=torch.zeros((1, 4), device="cuda").expand(4, 4))
    with pytest.raises(MvdbError):
        mx.product(p, p, out=torch.zeros((4, 4), device="cuda").t())
    for k in (0, -1, 129):
        with pytest.raises(MvdbError):
            mx.scan_many(p, p, k)
    with pytest.raises(MvdbError):
        mx.scan_many(p, p, 1, allow=torch.zeros((1,), dtype=torch.int64, device="cuda"))
    with pytest.raises(MvdbError):
        mx.scan_many(p, torch.zeros((40, 48), dtype=torch.uint8, device="cuda"), 1, allow=torch.zeros((1,), dtype=torch.int32, device="cuda"))
    with pytest.raises(MvdbError):
        mx.scan_many(p, p, 1, allow=torch.zeros((1,), dtype=torch.int32))
    torch.cuda.synchronize()


def test_empty_inputs(engines):
    import torch
    mx = engines(64)
    none = torch.zeros((0, 48), dtype=torch.uint8, device="cuda")
    some = mx.quantize(torch.randn((5, 64), device="cuda"))
    assert mx.quantize(torch.zeros((0, 64), device="cuda")).shape == (0, 48) and mx.expand(none).shape == (0, 64)
    assert mx.product(none, some).shape == (0, 5) and mx.product(some, none).shape == (5, 0)
    ids, val, cnt = mx.scan_many(none, some, 3)
    assert ids.shape == (0, 3) and cnt.shape == (0,)
    ids, val, cnt = mx.scan_many(some, none, 3)
    assert (ids == -1).all() and (val == 0).all() and (cnt == 0).all()


PRODUCT = [(1, 1), (1, 1000), (3, 64), (16, 129), (31, 33), (32, 4097), (33, 65), (64, 64), (100, 300), (129, 257), (300, 700), (513, 129)]


@pytest.mark.parametrize("nq,n", PRODUCT)
@pytest.mark.parametrize("dim", [4, 100, 384, 512])
def test_product_exact(engines, nq, n, dim):
    rng = np.random.default_rng(nq * 7 + n + dim)
    q, r = M.pack(_unit(rng, nq, dim)), M.pack(_unit(rng, n, dim))
    got = engines(dim).product(_to(q), _to(r)).cpu().numpy()
    want, _ = M.products(q, r, dim)
    assert np.array_equal(got.astype(np.float64), want)


@pytest.mark.parametrize("dim", [64, 68, 128, 192, 320, 448, 576, 640, 768, 1000, 1024, 1536, 4096])
def test_product_dimensions(engines, dim):
    rng = np.random.default_rng(dim)
    q, r = M.pack(_unit(rng, 70, dim)), M.pack(_unit(rng, 150, dim))
    got = engines(dim).product(_to(q), _to(r)).cpu().numpy().astype(np.float64)
    want, mag = M.products(q, r, dim)
    assert (np.abs(got - want) <= 65 * 2.0**-24 * (M.blocks(dim) // 2) * mag).all()


@pytest.mark.parametrize("dim", [64, 384, 1024])
def test_product_wide_scales_and_nan(engines, dim):
    rng = np.random.default_rng(dim)
    x = rng.standard_normal((90, dim)) * np.exp2(rng.integers(-20, 20, (90, dim)))
    y = rng.standard_normal((140, dim)) * np.exp2(rng.integers(-20, 20, (140, dim)))
    x[7, 3] = np.nan
    y[11, dim - 1] = np.inf
    q, r = M.pack(x.astype(np.float32)), M.pack(y.astype(np.float32))
    got = engines(dim).product(_to(q), _to(r)).cpu().numpy().astype(np.float64)
    want, mag = M.products(q, r, dim)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[7]).all() and np.isnan(got[:, 11]).all()
    fine = ~np.isnan(want)
    assert (np.abs(got - want)[fine] <= (65 * 2.0**-24 * (M.blocks(dim) // 2) * mag)[fine]).all()


def test_product_into_a_slice(engines):
    import torch
    rng = np.random.default_rng(5)
    q, r = M.pack(_unit(rng, 45, 384)), M.pack(_unit(rng, 130, 384))
    wide = torch.full((47, 200), -7.0, device="cuda")
    out = wide[1:46, 33:163]
    assert engines(384).product(_to(q), _to(r), out=out) is out
    got = wide.cpu().numpy()
    assert np.array_equal(got[1:46, 33:163].astype(np.float64), M.products(q, r, 384)[0])
    got[1:46, 33:163] = -7
    assert (got == -7).all()  # nothing around the slice was written


def _check_scan(mx, q, r, k, allow=None):
    """exact: sums representable in f32, so ids, values and counts are determined"""
    dim = mx.dim
    ids, val, cnt = mx.scan_many(_to(q), _to(r), k, None if allow is None else _to(allow.view(np.int32)))
    s, _ = M.products(q, r, dim)
    w_ids, w_val, w_cnt = M.topk(s, k, allow)
    assert np.array_equal(cnt.cpu().numpy(), w_cnt)
    assert np.array_equal(val.cpu().numpy().astype(np.float64), w_val)
    assert np.array_equal(ids.cpu().numpy(), w_ids)


def _bits(mask):
    n = mask.size
    w = np.zeros((n + 31) // 32 * 32, np.uint8)
    w[:n] = mask
    return np.packbits(w, bitorder="little").view(np.uint32)


SCAN = [(1, 1, 1, 64), (1, 5, 10, 64), (2, 63, 3, 100), (1, 5000, 10, 384), (5, 64, 128, 384), (17, 2049, 10, 384), (31, 3000, 1, 512),
        (33, 8191, 100, 100), (64, 20000, 10, 64), (65, 4500, 128, 384), (130, 9000, 32, 512), (257, 12345, 10, 384), (515, 7001, 12, 384),
        (3, 70000, 128, 64), (600, 40000, 10, 64), (40, 3001, 33, 1024), (300, 5003, 16, 1000), (9, 2500, 10, 640), (70, 66000, 7, 4)]


@pytest.mark.parametrize("nq,n,k,dim", SCAN)
def test_scan(engines, nq, n, k, dim):
    rng = np.random.default_rng(nq + n + k + dim)
    _check_scan(engines(dim), M.pack(_unit(rng, nq, dim)), M.pack(_unit(rng, n, dim)), k)


@pytest.mark.parametrize("share", [0.5, 0.03, 0.0005, 0.0])
@pytest.mark.parametrize("nq,n,k,dim", [(1, 9001, 10, 384), (40, 6007, 100, 100), (520, 20003, 10, 64)])
def test_scan_allow(engines, share, nq, n, k, dim):
    rng = np.random.default_rng(int(share * 10000) + nq)
    _check_scan(engines(dim), M.pack(_unit(rng, nq, dim)), M.pack(_unit(rng, n, dim)), k, _bits(rng.random(n) < share))


@pytest.mark.parametrize("nq", [1, 20, 300])
def test_scan_ties_and_duplicates(engines, nq):
    rng = np.random.default_rng(nq)
    base = _unit(rng, 50, 64)
    r = M.pack(base[rng.integers(0, 50, 6000)])  # every row about 120 times
    _check_scan(engines(64), M.pack(_unit(rng, nq, 64)), r, 100)
    same = np.repeat(M.pack(base[:1]), 30000, 0)  # one row over and over: the lowest ids
    _check_scan(engines(64), M.pack(_unit(rng, nq, 64)), same, 128)
    zero = np.zeros((3000, 64), np.float32)      # all products 0 (or -0): the lowest ids
    zero[::2] = -0.0
    _check_scan(engines(64), M.pack(_unit(rng, nq, 64)), M.pack(zero), 20)


@pytest.mark.parametrize("nq", [1, 40, 300])
@pytest.mark.parametrize("order", ["rising", "falling", "late block"])
def test_scan_ordered_rows(engines, nq, order):
    """Rows whose products with every query rise (each row beats all before it), fall, or are best in a few late blocks."""
    rng = np.random.default_rng(nq)
    n = 40000
    q = np.ones((nq, 64), np.float32) * np.exp2(rng.integers(-3, 3, (nq, 1))).astype(np.float32)
    at = np.arange(n)
    step = at // 2 if order == "rising" else (n - at) // 2 if order == "falling" else (at % 4096 >= 4000) * (1 + at % 77)

    def spell(t):  # 31 components that sum to t, each one a magnitude of the format
        j, rest = np.arange(31)[None, :], (t % 6)[:, None]
        full = (t // 6)[:, None]
        return np.where(j < full, 6, np.where(j == full, np.where(rest == 5, 4, rest), np.where((j == full + 1) & (rest == 5), 1, 0)))

    x = np.zeros((n, 64), np.float32)
    x[:, 0] = x[:, 32] = 6  # fixes the block's scale
    x[:, 1:32] = spell(step // 170)
    x[:, 33:] = spell(step % 170)
    x[:, 32:] /= 256
    assert np.array_equal(M.values(M.pack(x), 64), x)  # nothing is rounded: products rise with step
    r = M.pack(x)
    _check_scan(engines(64), M.pack(q), r, 100)


@pytest.mark.parametrize("nq,k", [(12, 10), (12, 100), (300, 10), (300, 100)])
def test_scan_adversarial_levels(engines, nq, k):
    """Rows in blocks of 64, every period-th block poor and the others good: where the period is that of a level, every row of
    the next beats the bound, more than any buffer holds."""
    rng = np.random.default_rng(3)
    n = 64 * 1500
    q = M.pack(np.ones((nq, 64)) + 0.5 * rng.integers(0, 2, (nq, 64)))
    for period in (2, 4, 5, 6, 7, 8, 10, 47, 49):
        good = (np.arange(n) // 64) % period != 0
        x = np.where(good[:, None], 1.0, -1.0) * (1 + 0.25 * rng.integers(0, 3, (n, 64)))
        _check_scan(engines(64), q, M.pack(x), k)


def test_scan_crowded_rows(engines):
    """Hundreds of neighbouring rows that are all candidates of one query (the chunks of one long document)."""
    rng = np.random.default_rng(4)
    x = _unit(rng, 50000, 64)
    q = _unit(rng, 30, 64)
    for i in range(30):
        at = 1000 + 1500 * i + 37 * i
        x[at : at + 20 * (i + 1)] = q[i] + 0.2 * rng.standard_normal((20 * (i + 1), 64)) / 8
    for nq in (1, 5, 30):
        _check_scan(engines(64), M.pack(q[-nq:]), M.pack(x), 128)
    _check_scan(engines(64), M.pack(np.repeat(q, 10, 0)), M.pack(x), 50)


def test_scan_many_queries(engines):
    """More queries than are dealt with at a time."""
    rng = np.random.default_rng(6)
    _check_scan(engines(64), M.pack(_unit(rng, 8200, 64)), M.pack(_unit(rng, 3300, 64)), 3)


@pytest.mark.parametrize("nq", [1, 70, 300])
def test_scan_leaves_out_nan(engines, nq):
    rng = np.random.default_rng(nq)
    x = _unit(rng, 5000, 100)
    x[rng.integers(0, 5000, 4000), rng.integers(0, 100, 4000)] = np.nan
    x[17, 40] = np.inf
    q = _unit(rng, nq, 100)
    _check_scan(engines(100), M.pack(q), M.pack(x), 50)
    q[0, 0] = np.nan  # a query that is not a number has no neighbours, the others keep theirs
    _check_scan(engines(100), M.pack(q), M.pack(x), 50)
    x[:] = np.nan
    _check_scan(engines(100), M.pack(_unit(rng, nq, 100)), M.pack(x), 5)


def test_scan_infinite_products(engines):
    """Products past the range of f32 are infinite and come first (or last), by id."""
    x = np.zeros((300, 64), np.float32)
    x[:, 0] = np.where(np.arange(300) % 3 == 0, 1e30, np.where(np.arange(300) % 3 == 1, -1e30, 1.0))
    q = np.zeros((2, 64), np.float32)
    q[:, 0] = [1e30, -1e30]
    ids, val, cnt = engines(64).scan_many(_to(M.pack(q)), _to(M.pack(x)), 128)
    v = val.cpu().numpy()
    assert (cnt.cpu().numpy() == 128).all() and np.isposinf(v[:, :100]).all() and np.isfinite(v[:, 100:]).all()
    assert np.array_equal(ids.cpu().numpy()[0, :100], np.arange(0, 300, 3)) and np.array_equal(ids.cpu().numpy()[1, :100], np.arange(1, 300, 3))
    for nq in (40, 300):  # in levels, the infinite ones late
        ids, val, cnt = engines(64).scan_many(_to(M.pack(np.repeat(q, nq // 2, 0))), _to(M.pack(np.concatenate([np.zeros((6000, 64), np.float32), x]))), 128)
        v, i = val.cpu().numpy(), ids.cpu().numpy()
        assert (cnt.cpu().numpy() == 128).all() and np.isposinf(v[:, :100]).all() and np.isfinite(v[:, 100:]).all()
        assert (i[: nq // 2, :100] == np.arange(6000, 6300, 3)).all() and (i[nq // 2 :, :100] == np.arange(6001, 6300, 3)).all()


@pytest.mark.parametrize("nq,n,dim", [(3, 4000, 384), (200, 9000, 1024)])
def test_scan_wide_scales(engines, nq, n, dim):
    """Where f32 sums round: the values are within the bound, and no row that is left out is clearly better than the last one."""
    rng = np.random.default_rng(n)
    mk = lambda m: M.pack((rng.standard_normal((m, dim)) * np.exp2(rng.integers(-16, 16, (m, dim)))).astype(np.float32))
    q, r = mk(nq), mk(n)
    k = 20
    ids, val, cnt = engines(dim).scan_many(_to(q), _to(r), k)
    ids, val = ids.cpu().numpy(), val.cpu().numpy().astype(np.float64)
    s, mag = M.products(q, r, dim)
    tol = 65 * 2.0**-24 * (M.blocks(dim) // 2) * mag
    assert (cnt.cpu().numpy() == k).all()
    for i in range(nq):
        assert len(set(ids[i])) == k and (np.diff(val[i]) <= 0).all()
        assert (np.abs(val[i] - s[i, ids[i]]) <= tol[i, ids[i]]).all()
        rest = np.ones(n, bool)
        rest[ids[i]] = False
        assert (s[i, rest] - tol[i, rest] <= val[i, -1]).all()


def test_scan_equals_product_topk_large(engines):
    """A million rows, on the device: the scan against the product it stands for."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    mx = engines(384)
    c = torch.randn((256, 384), generator=g, device="cuda")
    rows = mx.quantize(torch.nn.functional.normalize(c[torch.randint(0, 256, (1000000,), generator=g, device="cuda")]
                                                     + torch.randn((1000000, 384), generator=g, device="cuda")))
    q = mx.quantize(torch.nn.functional.normalize(c[torch.randint(0, 256, (1100,), generator=g, device="cuda")]
                                                  + torch.randn((1100, 384), generator=g, device="cuda")))
    for nq, k in ((1, 10), (24, 10), (24, 128), (1100, 10), (600, 128)):
        ids, val, cnt = mx.scan_many(q[:nq], rows, k)
        s = mx.product(q[:nq], rows)
        top = s.topk(k, dim=1).values
        assert torch.equal(val, top) and torch.equal(s.gather(1, ids.long()), val) and (cnt == k).all()
        tied = val[:, 1:] == val[:, :-1]
        assert (ids[:, 1:] > ids[:, :-1])[tied].all() and (torch.sort(ids, 1).values.diff(dim=1) > 0).all()
        # of the rows that tie with the last one the lowest ids were taken
        last = val[:, -1:]
        inside = (val == last).sum(1)
        for i in range(0, nq, max(1, nq // 50)):
            first = (s[i] == last[i]).nonzero().flatten()[: int(inside[i])]
            assert torch.equal(ids[i][val[i] == last[i]].long(), first)
        del s


def test_far_offsets(engines):
    """Packed rows and products whose offsets pass 32 bits."""
    import torch
    mx = engines(1024)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    n = 8_200_000  # x 544 B = 4.46 GB
    rows = torch.randint(0, 256, (n, 544), dtype=torch.uint8, device="cuda", generator=g)
    rows[:, 512:] = torch.randint(118, 122, (n, 32), dtype=torch.uint8, device="cuda", generator=g)
    q = rows[-70:].clone()  # their best rows are themselves, at the far end
    ids, val, cnt = mx.scan_many(q[:5], rows, 3)
    assert torch.equal(ids[:, 0].long(), torch.arange(n - 70, n - 65, device="cuda"))
    ids, val, cnt = mx.scan_many(q, rows, 3)
    assert torch.equal(ids[:, 0].long(), torch.arange(n - 70, n, device="cuda"))
    ids, val, cnt = mx.scan_many(q[:3], rows, 128)  # more keys than chunks may leave
    s3 = mx.product(q[:3], rows)
    assert torch.equal(val, s3.topk(128, dim=1).values) and torch.equal(s3.gather(1, ids.long()), val)
    del s3
    v = mx.expand(rows[-3000:])
    assert torch.equal(mx.quantize(v)[:, :512], mx.quantize(v.double().float())[:, :512])
    out = mx.product(rows[-300:], rows)  # 2.46e9 products
    want = mx.product(rows[-300:], rows[-500:].clone())
    assert torch.equal(out[:, -500:], want) and torch.equal(out[:, :200], mx.product(rows[-300:], rows[:200].clone()))
    del out
    x = mx.expand(rows[:1_100_000])  # 4.5 GB of f32
    assert torch.equal(mx.expand(mx.quantize(x)), x)
    one = x[-2:].clone()
    assert torch.equal(mx.quantize(x)[-2:], mx.quantize(one))


def test_graph_capture(engines):
    """quantise -> scan and product in one graph, replayed with other inputs, eager calls of the same kind in between."""
    import torch
    mx = engines(384)
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    rows = mx.quantize(torch.randn((30000, 384), generator=g, device="cuda"))
    for nq in (1, 300):
        x = torch.randn((nq, 384), generator=g, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            mx.scan_many(mx.quantize(x), rows, 10)
        torch.cuda.current_stream().wait_stream(side)
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p = mx.quantize(x)
            got = mx.scan_many(p, rows, 10)
            scores = mx.product(p, rows[:500])
        with torch.cuda.graph(other):  # a second one, with a workspace of its own
            got2 = mx.scan_many(mx.quantize(x), rows, 100)
        for rep in range(4):
            x.copy_(torch.randn((nq, 384), generator=g, device="cuda"))
            graph.replay()
            other.replay()
            torch.cuda.synchronize()
            want, want2 = mx.scan_many(mx.quantize(x), rows, 10), mx.scan_many(mx.quantize(x), rows, 100)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(got2, want2))
            assert torch.equal(scores, mx.product(mx.quantize(x), rows[:500]))


@pytest.mark.parametrize("nq", [1, 40, 300])
def test_capture_without_a_call_before(gpu, nq):
    """A handle and a row length that nothing has used yet: the first call of all may be the captured one."""
    import torch
    from minivectordb_amd import HipBridge
    from minivectordb_amd.pipeline import ResidentMx4
    dim = {1: 708, 40: 836, 300: 900}[nq]
    b = HipBridge(device=0)
    b.init(dict(dim=dim, m=8, ef=50, capacity=8, seed=1))
    mx = ResidentMx4(b, torch.device("cuda", 0))
    rng = np.random.default_rng(nq)
    q, r = M.pack(_unit(rng, nq, dim)), M.pack(_unit(rng, 5000, dim))
    qd, rd = _to(q), _to(r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mx.scan_many(qd, rd, 10)
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(got[0].cpu().numpy(), M.topk(M.products(q, r, dim)[0], 10)[0])
    del graph
    b.close()


def test_streams_side_by_side(engines):
    import torch
    mx = engines(384)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    rows = mx.quantize(torch.randn((50000, 384), generator=g, device="cuda"))
    qs = [mx.quantize(torch.randn((n, 384), generator=g, device="cuda")) for n in (1, 700, 40, 700, 5, 64)]
    want = [mx.scan_many(q, rows, 20) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(3):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(mx.scan_many(q, rows, 20))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_workspace_is_caller_owned(engines):
    """The C entry point with a workspace full of other bytes, just as long as asked for; nothing behind it is written."""
    import torch
    mx = engines(100)
    rng = np.random.default_rng(0)
    for nq, n, k in ((1, 3000, 10), (90, 5000, 128), (600, 3000, 5)):
        q, r = M.pack(_unit(rng, nq, 100)), M.pack(_unit(rng, n, 100))
        need = mx.L.mvdb_mx4_scan_workspace(mx.b.handle, nq, n, k)
        for fill in (0, 0xFF, 0x7F):
            ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device="cuda")
            ids = torch.full((nq, k), -5, dtype=torch.int32, device="cuda")
            val = torch.full((nq, k), -5.0, device="cuda")
            cnt = torch.full((nq,), -5, dtype=torch.int32, device="cuda")
            qd, rd, vp = _to(q), _to(r), C.c_void_p
            ok = mx.L.mvdb_mx4_scan_many_dev(mx.b.handle, vp(qd.data_ptr()), nq, vp(rd.data_ptr()), n, k, None, vp(ids.data_ptr()),
                                             vp(val.data_ptr()), vp(cnt.data_ptr()), vp(ws.data_ptr()), need,
                                             vp(torch.cuda.current_stream().cuda_stream))
            assert ok == 1, mx.L.mvdb_last_error(mx.b.handle)
            torch.cuda.synchronize()
            assert (ws[need:] == fill).all()
            w = M.topk(M.products(q, r, 100)[0], k)
            assert np.array_equal(ids.cpu().numpy(), w[0]) and np.array_equal(cnt.cpu().numpy(), w[2])


def test_host_forms_and_rerank(engines):
    """The run of them a search makes from host buffers: attach, scan for candidates with a filter, rerank on the f32 store."""
    from minivectordb_amd import HipBridge
    rng = np.random.default_rng(21)
    n, dim, nq, k, topk = 20000, 384, 50, 100, 10
    base, q = _unit(rng, n, dim), _unit(rng, nq, dim)
    b = HipBridge(device=0)
    b.init(dict(dim=dim, m=8, ef=50, capacity=n, seed=1))
    packed, vals = b.mx4Quantize(base[:777])
    assert np.array_equal(packed, M.pack(base[:777])) and np.array_equal(vals, M.values(packed, dim).astype(np.float32))
    b.mx4Attach(base)
    assert b.mx4Rows() == n
    s, _ = M.products(M.pack(q), M.pack(base), dim)
    assert np.array_equal(b.mx4ProductMany(q).astype(np.float64), s)
    allow = _bits(rng.random(n) < 0.4)
    ids, val, cnt = b.mx4ScanMany(q, k, allow)
    w_ids, w_val, w_cnt = M.topk(s, k, allow)
    assert np.array_equal(ids, w_ids) and np.array_equal(val.astype(np.float64), w_val) and np.array_equal(cnt, w_cnt)
    b.attachF32(base, resident=True)
    r_ids, r_l2, r_n = b.rerankMany(q, ids, cnt, k, topk, allow)
    d = np.square(q[:, None, :].astype(np.float64) - base[w_ids].astype(np.float64)).sum(-1)
    for i in range(nq):
        order = np.lexsort((w_ids[i], d[i]))[:topk]
        assert np.array_equal(r_ids[i], w_ids[i][order]) and r_n[i] == topk
    # 100 candidates of 4 bits hold nearly all of the true ten (allowed rows, f32)
    ok = ((allow[np.arange(n) >> 5] >> (np.arange(n) & 31).astype(np.uint32)) & 1).astype(bool)
    true = np.argsort(np.where(ok, np.square(q[:, None].astype(np.float32) - base[None]).sum(-1), np.inf), 1)[:, :topk]
    assert np.mean([len(set(t) & set(g)) / topk for t, g in zip(true, r_ids)]) > 0.9
    b.mx4Attach(base[:100])
    assert b.mx4Rows() == 100 and b.mx4ScanMany(q[:2], 128)[2].tolist() == [100, 100]
    b.mx4Attach(None)
    assert b.mx4Rows() == 0
    b.close()


def test_database_candidates(gpu, tmp_path):
    """MiniVectorDB.searchMany({"candidates": "mx4"}): the four operators' run under the facade, with a filter, deletions, later
    inserts and a reopened store."""
    from minivectordb_amd import MiniVectorDB
    rng = np.random.default_rng(8)
    n, dim = 3000, 100
    x = _unit(rng, n + 50, dim)
    q = _unit(rng, 20, dim)
    db = MiniVectorDB.open(dict(storageDir=str(tmp_path), dim=dim, capacity=8000, seed=1, preloadVectors=True))
    assert db.searchMany(q, {"topK": 3, "candidates": "mx4"}) == [[]] * 20
    db.insertMany([dict(id=f"d{i}", input=x[i], metadata=dict(kind=i % 3)) for i in range(n)])

    def true(rows):  # ids of the nearest among `rows`, and their distances, in 64 bits from the normalised rows
        xn = x[rows].astype(np.float64) / np.linalg.norm(x[rows].astype(np.float64), axis=1, keepdims=True)
        qn = q.astype(np.float64) / np.linalg.norm(q.astype(np.float64), axis=1, keepdims=True)
        d = np.square(qn[:, None] - xn[None]).sum(-1)
        o = np.argsort(d, 1, kind="stable")
        return np.asarray(rows)[o], np.take_along_axis(d, o, 1)

    def check(got, rows, topk):
        ids, d = true(rows)
        hits = 0
        for i in range(20):
            assert len(got[i]) == min(topk, len(rows))
            by = {f"d{j}": v for j, v in zip(ids[i], d[i])}
            for r in got[i]:  # what comes back is allowed, in order, and at its f32 distance
                assert abs(by[r["id"]] - r["score"]) <= 1e-5
            assert [r["score"] for r in got[i]] == sorted(r["score"] for r in got[i])
            hits += len({r["id"] for r in got[i]} & {f"d{j}" for j in ids[i][:topk]})
        assert hits >= 0.95 * 20 * min(topk, len(rows))  # 128 candidates of 4 bits for the best `topk`

    check(db.searchMany(q, {"topK": 10, "candidates": "mx4"}), list(range(n)), 10)
    check(db.searchMany(q, {"topK": 10, "candidates": "mx4", "filter": {"kind": 1}}), list(range(1, n, 3)), 10)
    db.removeMany([f"d{i}" for i in range(0, n, 2)])
    check(db.searchMany(q, {"topK": 5, "candidates": "mx4"}), list(range(1, n, 2)), 5)
    db.insertMany([dict(id=f"d{i}", input=x[i], metadata=dict(kind=7)) for i in range(n, n + 50)])
    check(db.searchMany(q, {"topK": 60, "candidates": "mx4", "filter": {"kind": 7}}), list(range(n, n + 50)), 60)
    assert db.searchMany([x[n + 7]], {"topK": 1, "candidates": "mx4"})[0][0]["id"] == f"d{n + 7}"
    db.save()
    db.close()
    db = MiniVectorDB.open(dict(storageDir=str(tmp_path), dim=dim, capacity=8000, seed=1, preloadVectors=False))
    check(db.searchMany(q, {"topK": 10, "candidates": "mx4", "filter": {"kind": 7}}), list(range(n, n + 50)), 10)
    with pytest.raises(Exception, match="at most 128"):
        db.searchMany(q, {"topK": 129, "candidates": "mx4"})
    with pytest.raises(ValueError, match="candidates"):
        db.searchMany(q, {"topK": 1, "candidates": "mx5"})
    db.close()
    db.init()  # the same object on a new engine, which holds neither store of rows
    check(db.searchMany(q, {"topK": 10, "candidates": "mx4", "filter": {"kind": 7}}), list(range(n, n + 50)), 10)
    db.close()
