"""Products of microscaled 4-bit rows at both ends of f32's range, and far ends of large stores, against the 64-bit oracle.

Tolerance at the small end.  A matrix instruction adds 64 products and the accumulator, each cut at 2^-24 of the largest of them or at the
least f32 there is, 2^-149, whichever is more; so with P = sum |q_i r_i| the error is at most 65 (2^-24 P + 2^-149) for each of dim / 64
instructions."""
import numpy as np
import pytest

from oracle import mx4_oracle as M
from test_gpu_mx4_lengths import engines  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def _to(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("low", [-62, -68, -72, -75, -80])
@pytest.mark.parametrize("dim", [64, 384, 1000, 2048])
def test_product_of_small_values(engines, dim, low):
    """Results down to the least f32 and below."""
    rng = np.random.default_rng(dim - low)
    mk = lambda n: M.pack((rng.standard_normal((n, dim)) * np.exp2(low + rng.integers(-2, 3, (n, dim)))).astype(np.float32))
    q, r = mk(40), mk(70)
    got = engines(dim).product(_to(q), _to(r)).cpu().numpy().astype(np.float64)
    want, mag = M.products(q, r, dim)
    assert (np.abs(got - want) <= 65 * (M.blocks(dim) // 2) * (2.0**-24 * mag + 2.0**-149)).all()
    if low > -72:
        assert (got != 0).mean() > 0.9  # nothing is taken for 0 that is not


@pytest.mark.parametrize("dim", [64, 128, 384, 1000, 2048])
def test_product_of_large_values(engines, dim):
    """Sums whose terms' magnitudes add up to more than f32 holds: infinite where the terms have one sign; where they do not the
    sum itself, or infinite (a part of it passed the range); never not a number."""
    x = np.zeros((8, dim), np.float32)
    y = np.zeros((4, dim), np.float32)
    big = np.float32(2.0**100)
    y[0, :] = big
    y[1, :] = -big
    y[2, :] = np.where(np.arange(dim) % 2, big, -big)
    y[3, :2] = big
    x[0, 0] = big                                            # past the range in the first group
    x[1, dim - 1] = -big                                     # in the last
    x[2, [0, 1]] = big, -big                                 # cancels within a group
    x[3, 0], x[3, dim - 1] = big, -big                       # cancels: within a group where there is one, else after the infinity
    x[4, 0], x[4, dim - 1] = -big, big
    x[5, 0] = 2.0**20                                        # 2^120: fits
    x[6, 0], x[6, 1] = 2.0**27, -(2.0**27)                   # 2^127 - 2^127
    x[7] = 3e38
    got = engines(dim).product(_to(M.pack(x)), _to(M.pack(y))).cpu().numpy().astype(np.float64)
    _check_large(got, M.values(M.pack(x), dim), M.values(M.pack(y), dim))


@pytest.mark.parametrize("dim", [64, 128, 1000, 2048])
def test_product_of_largest_values(engines, dim):
    rng = np.random.default_rng(dim)
    x = (3.4e38 * rng.choice([-1.0, 1.0, 0.0], (40, dim))).astype(np.float32)
    x[0], x[1], x[2] = 3.4e38, -3.4e38, 0
    p = M.pack(x)
    got = engines(dim).product(_to(p), _to(p)).cpu().numpy().astype(np.float64)
    _check_large(got, M.values(p, dim), M.values(p, dim))


def _check_large(got, v, w):
    top = float(np.finfo(np.float32).max)
    want, mag = v @ w.T, np.abs(v) @ np.abs(w).T
    assert not np.isnan(got).any()
    fits = mag <= top
    assert np.array_equal(got[fits], want[fits]) and fits.any()
    one_sign = ~fits & (np.abs(want) == mag)
    assert np.array_equal(got[one_sign], np.sign(want[one_sign]) * np.inf) and one_sign.any()
    rest = ~fits & ~one_sign  # the sum itself, or infinite
    with np.errstate(over="ignore"):
        as32 = want.astype(np.float32).astype(np.float64)
    assert (np.isinf(got) | (got == as32))[rest].all()


def test_far_ends_of_large_stores(engines):
    """Expansion and quantisation where offsets pass 32 bits (packed rows of 4.46 GB, values of 4.5 GB), against the oracle."""
    import torch
    mx = engines(1024)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    n = 8_200_000
    rows = torch.randint(0, 256, (n, 544), dtype=torch.uint8, device="cuda", generator=g)
    rows[:, 512:] = torch.randint(118, 122, (n, 32), dtype=torch.uint8, device="cuda", generator=g)
    tail = mx.expand(rows[-3000:])  # packed rows past 4 GB
    assert np.array_equal(tail.cpu().numpy(), M.values(rows[-3000:].cpu().numpy(), 1024).astype(np.float32))
    m = 1_100_000
    x = mx.expand(rows[:m])  # values past 4 GB
    for at in (slice(0, 500), slice(m // 2, m // 2 + 500), slice(m - 500, m)):
        assert np.array_equal(x[at].cpu().numpy(), M.values(rows[at].cpu().numpy(), 1024).astype(np.float32))
    del rows
    x[-500:] = torch.randn((500, 1024), generator=g, device="cuda")
    p = mx.quantize(x)
    assert np.array_equal(p[-500:].cpu().numpy(), M.pack(x[-500:].cpu().numpy()))
    del p
    wide = torch.zeros((4_200_000, 1030), dtype=torch.float16, device="cuda")  # rows apart, 8.6 GB from the first to the last; more than 2^22 of them
    wide[-300:, 3:1027] = torch.randn((300, 1024), generator=g, device="cuda").half()
    p = mx.quantize(wide[:, 3:1027])
    assert np.array_equal(p[-300:].cpu().numpy(), M.pack(wide[-300:, 3:1027].double().cpu().numpy()))
    assert not p[:-300].any()
