"""Microscaled 4-bit operators without a GPU: the oracle on known answers, and what every entry point refuses before it
touches a device."""
import ctypes as C

import numpy as np
import pytest

from minivectordb_amd import HipBridge, MvdbError
from oracle import mx4_oracle as M


def _bridge(dim):
    b = HipBridge()
    b.init(dict(dim=dim, m=8, ef=50, capacity=8, seed=1))
    return b


def test_oracle_known_answers():
    x = np.zeros((1, 64))
    x[0, :8] = [6, 4, -3, 2, 1.5, -1, 0.5, 0.25]          # largest 6: scale 2^0; 0.25 is a tie, to the even code 0
    x[0, 32:40] = [7.9, 5, 3.5, 2.5, 1.75, 1.25, 0.75, -5]  # ties: 5 -> 4, 3.5 -> 4, 2.5 -> 2, 1.75 -> 2, 1.25 -> 1, 0.75 -> 1
    code, s = M.codes_and_scales(x)
    assert s.tolist() == [[127, 127]]
    assert code[0, 0, :8].tolist() == [7, 6, 13, 4, 3, 10, 1, 0]
    assert code[0, 1, :8].tolist() == [7, 6, 6, 4, 4, 2, 2, 14]
    p = M.pack(x)
    assert p.shape == (1, 48) and p[0, 0] == 7 | (6 << 4) and p[0, 32:34].tolist() == [127, 127] and not p[0, 34:].any()
    assert M.values(p, 64)[0, :8].tolist() == [6, 4, -3, 2, 1.5, -1, 0.5, 0]


def test_oracle_scales():
    x = np.zeros((6, 64))
    x[0, 0] = 2.0**-126   # floor(log2) - 2 below -127: the scale stays there
    x[1, 0] = 2.0**-149
    x[2, 0] = np.float32(3.4028235e38)
    x[3, 0] = 8.0         # 8 = 4 * 2^1
    x[4, 0] = np.nextafter(np.float32(8), np.float32(0))
    x[5, 0] = np.inf
    code, s = M.codes_and_scales(x)
    assert s[:, 0].tolist() == [0, 0, 252, 128, 127, 255] and s[:, 1].tolist() == [0] * 6
    assert code[:, 0, 0].tolist() == [4, 0, 7, 6, 7, 0]
    assert M.values(M.pack(x), 64)[0, 0] == 2.0**-126 and np.isnan(M.values(M.pack(x), 64)[5, 0])


def test_oracle_topk_order():
    s = np.array([[1.0, 2.0, np.nan, 2.0, -0.0, 0.0]])
    assert M.topk(s, 4)[0].tolist() == [[1, 3, 0, 4]]
    ids, val, cnt = M.topk(s, 4, np.array([0b110100], np.uint32))
    assert ids.tolist() == [[4, 5, -1, -1]] and cnt.tolist() == [2]


@pytest.mark.parametrize("dim,want", [(4, 48), (64, 48), (68, 80), (384, 208), (512, 272), (516, 320), (1000, 544), (1024, 544)])
def test_row_bytes(dim, want):
    b = _bridge(dim)
    assert b.mx4RowBytes() == want == M.row_bytes(dim)
    b.close()


def _refused(b, ok, text):
    assert ok == 0 and text in b._L.mvdb_last_error(b.handle).decode(), b._L.mvdb_last_error(b.handle)


def test_device_entry_points_refuse():
    """Addresses are only looked at, never followed: every call here is refused before a device is needed."""
    b = _bridge(64)
    L, h, vp = b._L, b.handle, C.c_void_p
    a = vp(1 << 20)  # aligned, never followed
    q = lambda *x: L.mvdb_mx4_quantize_dev(h, *x, None)
    _refused(b, q(a, 3, 1, 64, a), "dtype")
    _refused(b, q(a, 0, -1, 64, a), "negative")
    _refused(b, q(a, 0, 1, 63, a), "ld is smaller")
    _refused(b, q(None, 0, 1, 64, a), "null")
    _refused(b, q(a, 0, 1, 64, None), "null")
    _refused(b, q(vp((1 << 20) + 2), 0, 1, 64, a), "aligned")
    _refused(b, q(vp((1 << 20) + 1), 1, 1, 64, a), "aligned")
    _refused(b, q(a, 0, 1, 64, vp((1 << 20) + 8)), "16-byte")
    assert q(None, 0, 0, 64, None) == 1
    e = lambda *x: L.mvdb_mx4_expand_dev(h, *x, None)
    _refused(b, e(a, -1, a), "negative")
    _refused(b, e(None, 1, a), "null")
    _refused(b, e(vp((1 << 20) + 4), 1, a), "16-byte")
    _refused(b, e(a, 1, vp((1 << 20) + 2)), "aligned")
    assert e(None, 0, None) == 1
    p = lambda *x: L.mvdb_mx4_product_dev(h, *x, None)
    _refused(b, p(a, -1, a, 1, a, 1), "negative")
    _refused(b, p(a, 1, a, -1, a, 1), "negative")
    _refused(b, p(a, 2, a, 5, a, 4), "ldo")
    _refused(b, p(a, 2, None, 5, a, 5), "null")
    _refused(b, p(vp((1 << 20) + 8), 2, a, 5, a, 5), "16-byte")
    _refused(b, p(a, 2, a, 5, vp((1 << 20) + 2), 5), "aligned")
    assert p(None, 0, None, 5, None, 5) == 1 and p(None, 5, None, 0, None, 0) == 1
    ws = L.mvdb_mx4_scan_workspace(h, 3, 100, 10)
    assert ws > 0 and L.mvdb_mx4_scan_workspace(h, 3, 100, 129) == 0 and L.mvdb_mx4_scan_workspace(h, 3, -1, 10) == 0
    s = lambda nq, n, k, w, z, qq=a, rr=a: L.mvdb_mx4_scan_many_dev(h, qq, nq, rr, n, k, None, a, a, a, w, z, None)
    _refused(b, s(3, 100, 0, a, ws), "k must be")
    _refused(b, s(3, 100, 129, a, 1 << 30), "k must be")
    _refused(b, s(-3, 100, 10, a, ws), "negative")
    _refused(b, s(3, -100, 10, a, ws), "negative")
    _refused(b, s(3, 100, 10, None, ws), "null")
    _refused(b, s(3, 100, 10, a, ws - 1), "workspace is smaller")
    _refused(b, s(3, 100, 10, vp((1 << 20) + 4), ws), "workspace must be 16-byte")
    _refused(b, s(3, 100, 10, a, ws, vp((1 << 20) + 4)), "packed rows must be 16-byte")
    _refused(b, s(3, 100, 10, a, ws, a, None), "null")
    _refused(b, L.mvdb_mx4_scan_many_dev(h, a, 3, a, 100, 10, vp((1 << 20) + 2), a, a, a, a, ws, None), "filter is not aligned")
    assert s(0, 100, 10, None, 0, None, None) == 1
    b.close()


def test_dimensions_refused():
    b = _bridge(4100)
    a = C.c_void_p(1 << 20)
    _refused(b, b._L.mvdb_mx4_quantize_dev(b.handle, a, 0, 1, 4100, a, None), "dim > 4096")
    _refused(b, b._L.mvdb_mx4_expand_dev(b.handle, a, 1, a, None), "dim > 4096")
    _refused(b, b._L.mvdb_mx4_product_dev(b.handle, a, 1, a, 1, a, 1, None), "dim > 4096")
    b.close()
    b = _bridge(1028)
    _refused(b, b._L.mvdb_mx4_scan_many_dev(b.handle, a, 1, a, 1, 1, None, a, a, a, a, 1 << 20, None), "dim > 1024")
    b.close()


def test_host_entry_points_refuse():
    b = _bridge(64)
    x = np.zeros((2, 64), np.float32)
    assert b.mx4Rows() == 0
    with pytest.raises(MvdbError, match="no 4-bit store"):
        b.mx4ScanMany(x, 5)
    for k in (0, 129, 1 << 40):  # refused before anything of that size is made
        with pytest.raises(MvdbError, match="k must be 1..128"):
            b.mx4ScanMany(x, k)
    with pytest.raises(MvdbError, match="no 4-bit store"):
        b.mx4ProductMany(x)
    with pytest.raises(MvdbError, match="dim"):
        b.mx4Quantize(np.zeros((2, 60), np.float32))
    with pytest.raises(MvdbError, match="dim"):
        b.mx4Attach(np.zeros((2, 60), np.float32))
    _refused(b, b._L.mvdb_mx4_attach(b.handle, None, -1), "out of range")
    _refused(b, b._L.mvdb_mx4_attach(b.handle, None, 1 << 31), "out of range")
    _refused(b, b._L.mvdb_mx4_quantize(b.handle, None, 1, None, None), "null")
    b.close()


def test_resident_refuses():
    import torch
    from minivectordb_amd.pipeline import ResidentMx4
    b = _bridge(64)
    with pytest.raises(MvdbError, match="GPU device"):
        ResidentMx4(b, torch.device("cpu"))
    with pytest.raises(MvdbError, match="works on cuda:0"):
        ResidentMx4(b, torch.device("cuda", 1))
    mx = ResidentMx4(b, torch.device("cuda", 0))
    with pytest.raises(MvdbError, match="cuda:0"):
        mx.quantize(torch.zeros((2, 64)))
    with pytest.raises(MvdbError, match="cuda:0"):
        mx.expand(torch.zeros((2, 48), dtype=torch.uint8))
    with pytest.raises(MvdbError, match="cuda:0"):
        mx.product(torch.zeros((2, 48), dtype=torch.uint8), torch.zeros((2, 48), dtype=torch.uint8))
    with pytest.raises(MvdbError, match="cuda:0"):
        mx.scan_many(torch.zeros((2, 48), dtype=torch.uint8), torch.zeros((2, 48), dtype=torch.uint8), 3)
    with pytest.raises(MvdbError, match="cuda:0"):
        mx.quantize("rows")
    b.close()
    with pytest.raises(MvdbError, match="not initialized"):
        mx.row_bytes
