"""What the 4-bit store's host entry points refuse, without a GPU."""
from minivectordb_amd import HipBridge


def test_attach_refuses_rows_without_an_address():
    """A null address with rows is a mistake of the caller's, not a request to drop the store."""
    b = HipBridge()
    b.init(dict(dim=64, m=8, ef=50, capacity=8, seed=1))
    assert b._L.mvdb_mx4_attach(b.handle, None, 5) == 0
    assert "mvdb_mx4_attach: null pointer" in b._L.mvdb_last_error(b.handle).decode()
    b.close()


def test_scan_workspace_follows_the_store():
    """A scan's workspace is no larger than the lists that its rows can fill."""
    b = HipBridge()
    b.init(dict(dim=64, m=8, ef=50, capacity=8, seed=1))
    ws = lambda nq, n, k: b._L.mvdb_mx4_scan_workspace(b.handle, nq, n, k)
    for nq, k in ((300, 10), (300, 128), (512, 10), (1000, 10), (4096, 100)):
        sizes = [ws(nq, n, k) for n in (0, 64, 2048, 2049, 5000, 10000, 20000, 1 << 20)]
        assert min(sizes) > 0
        # 64 rows are a tile; a workgroup takes at least one, and leaves two lists a query, here of at most 128 records of 20 bytes
        for n, size in zip((0, 64, 2048, 2049, 5000, 10000, 20000), sizes):
            tiles = (n + 63) // 64
            assert size <= nq * (2 * (tiles + 8) * (128 * 20 + 4) + 2048) + 4096
    assert ws(300, 5000, 10) < 40 << 20
    b.close()
