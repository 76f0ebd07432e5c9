"""The scan of microscaled 4-bit rows at every row length its kernels are made for (1 .. 16 steps of 64 components), against sums
in 64 bits and a stable sort on the GPU.

The reference: `expand` (every value of which is tested against the oracle elsewhere) -> float64 -> one matrix product, sorted by (value
descending, id ascending).  No tolerance: unit rows have scales that lie within a few powers of two, and their f32 sums are
exact (a product is a multiple of 1/4 of its two scales' product and at most 36 of it, so sums over dim components whose
scales' products span 2^w need 2 + log2(36 dim) + w <= 24 bits; the test computes w from the packed rows and asserts it)."""
import numpy as np
import pytest

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


def unit_rows(g, n, dim):
    import torch
    c = torch.randn((64, dim), generator=g, device="cuda")
    x = c[torch.randint(0, 64, (n,), generator=g, device="cuda")] + torch.randn((n, dim), generator=g, device="cuda")
    return torch.nn.functional.normalize(x)


def random_bits(g, n, share):
    """-> (bitmap words, which rows pass)"""
    import torch
    bits = torch.rand(((n + 31) // 32, 32), generator=g, device="cuda") < share
    words = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    return words, bits.flatten()[:n]


def scales_spread(mx, q, r):
    """log2 of the spread of the products of two scales (blocks of zeros do not count)"""
    nb = 2 * ((mx.dim + 63) // 64)
    spread = 0
    for p in (q, r):
        s = p[:, 16 * nb : 17 * nb].int()
        spread += int(s.max()) - int(s.masked_fill(s == 0, 255).min())
    return spread


def want_scan(mx, q, r, k, keep=None, exact=True):
    """(ids, values, counts) of the k best, from 64-bit sums"""
    import torch
    if exact:
        assert 2 + np.log2(36 * mx.dim) + scales_spread(mx, q, r) <= 24
    rt = mx.expand(r).double().T.contiguous()
    ids, val, cnt = [], [], []
    for part in torch.split(mx.expand(q).double(), 512):
        s = part @ rt
        s += 0.0  # -0 is 0
        s = s.masked_fill(torch.isnan(s), -float("inf"))
        if keep is not None:
            s = s.masked_fill(~keep, -float("inf"))
        if s.shape[1] < k:
            s = torch.nn.functional.pad(s, (0, k - s.shape[1]), value=-float("inf"))
        v, i = torch.sort(s, dim=1, descending=True, stable=True)
        v, i = v[:, :k], i[:, :k]
        got = v > -float("inf")
        ids.append(torch.where(got, i, -1).int())
        val.append(torch.where(got, v, 0.0))
        cnt.append(got.sum(1).int())
    return torch.cat(ids), torch.cat(val), torch.cat(cnt)


def check(got, want):
    import torch
    assert torch.equal(got[2], want[2])
    assert torch.equal(got[1].double(), want[1])
    assert torch.equal(got[0], want[0])


# steps of 64 components; 300 queries: a workgroup a selection, 8 to 9 tiles a workgroup; 2200 queries: 10 tiles a workgroup, a wave a
# selection (k 10) and a workgroup a selection (k 100)
@pytest.mark.parametrize("share", [1.0, 0.3])
@pytest.mark.parametrize("nq,n,k", [(300, 140003, 10), (2200, 30011, 10), (2200, 30011, 100), (40, 60013, 10), (5, 60013, 20)])
@pytest.mark.parametrize("steps", range(1, 17))
def test_scan_every_length(engines, steps, nq, n, k, share):
    import torch
    dim = 64 * steps - 4 * (steps % 5)  # ends inside a block, or not
    g = torch.Generator(device="cuda")
    g.manual_seed(1000 * steps + nq + k)
    mx = engines(dim)
    q, r = mx.quantize(unit_rows(g, nq, dim)), mx.quantize(unit_rows(g, n, dim))
    words, keep = random_bits(g, n, share) if share < 1 else (None, None)
    check(mx.scan_many(q, r, k, words), want_scan(mx, q, r, k, keep))
