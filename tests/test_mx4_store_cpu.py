"""What the 4-bit store's host entry points refuse, without a GPU."""
from minivectordb_amd import HipBridge


def test_attach_refuses_rows_without_an_address():
    """A null address with rows is a mistake of the caller's, not a request to drop the store."""
    b = HipBridge()
    b.init(dict(dim=64, m=8, ef=50, capacity=8, seed=1))
    assert b._L.mvdb_mx4_attach(b.handle, None, 5) == 0
    assert "mvdb_mx4_attach: null pointer" in b._L.mvdb_last_error(b.handle).decode()
    b.close()
