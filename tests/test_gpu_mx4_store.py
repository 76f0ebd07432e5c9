"""The 4-bit store that a handle keeps (mvdb_mx4_attach), and the memory that it takes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _bridge(dim):
    from minivectordb_amd import HipBridge
    b = HipBridge(device=0)
    b.init(dict(dim=dim, m=8, ef=50, capacity=8, seed=1))
    return b


def _free():
    import torch
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def test_store_gives_its_memory_back(gpu):
    """A store that is dropped, or takes the place of a much larger one, frees what it held: 96 MB here."""
    b = _bridge(64)
    x = np.random.default_rng(0).standard_normal((2_000_000, 64), dtype=np.float32)
    b.mx4Attach(x)
    assert b.mx4Rows() == len(x)
    held = _free()
    b.mx4Attach(x[:1000])
    assert b.mx4Rows() == 1000 and _free() >= held + (90 << 20)
    want = b.mx4ScanMany(x[:3], 5)
    assert (want[0][:, 0] == [0, 1, 2]).all()
    b.mx4Attach(x)
    held = _free()
    b.mx4Attach(None)
    assert b.mx4Rows() == 0 and _free() >= held + (90 << 20)
    b.mx4Attach(x[:1000])  # and it can be filled again
    got = b.mx4ScanMany(x[:3], 5)
    assert all(np.array_equal(a, c) for a, c in zip(got, want))
    b.close()


def test_refused_attach_keeps_the_store(gpu):
    b = _bridge(64)
    x = np.random.default_rng(1).standard_normal((100, 64), dtype=np.float32)
    b.mx4Attach(x)
    assert b._L.mvdb_mx4_attach(b.handle, None, 5) == 0 and b._L.mvdb_mx4_attach(b.handle, None, -1) == 0
    assert b.mx4Rows() == 100 and (b.mx4ScanMany(x[:3], 5)[0][:, 0] == [0, 1, 2]).all()
    b.close()


def test_host_product_keeps_little_memory(gpu):
    """The handle keeps its staging of products between calls: 256 MB at most, and as much of f32 rows, however many products a call makes."""
    b = _bridge(64)
    x = np.random.default_rng(2).standard_normal((500_000, 64), dtype=np.float32)
    b.mx4Attach(x)
    b.mx4ProductMany(x[:1])  # (code and queries on the device)
    held = _free()
    out = b.mx4ProductMany(x[:300])  # 600 MB of products
    assert held - _free() <= 260 << 20
    assert np.array_equal(out[:140], b.mx4ProductMany(x[:140])) and np.array_equal(out[140:], b.mx4ProductMany(x[140:300]))
    b.close()


def test_database_opened_with_less_room(gpu, tmp_path):
    """A store of 300 vectors opened again with room for 100: both kinds of candidates answer from the vectors that there is room for."""
    from minivectordb_amd import MiniVectorDB
    x = np.random.default_rng(0).standard_normal((300, 64)).astype(np.float32)
    opts = dict(storageDir=str(tmp_path), dim=64, seed=1, preloadVectors=True)
    db = MiniVectorDB.open(dict(opts, capacity=300))
    db.insertMany([dict(id=f"d{i}", input=v) for i, v in enumerate(x)])
    db.close()  # (without a snapshot of the graph, which would keep its room)
    db = MiniVectorDB.open(dict(opts, capacity=100))
    assert db.wasm.getMaxElements() == 100
    xn = x.astype(np.float64) / np.linalg.norm(x.astype(np.float64), axis=1, keepdims=True)
    for at in (3, 99, 250):
        want = [f"d{i}" for i in np.argsort(np.square(xn[at] - xn[:100]).sum(1), kind="stable")[:5]]
        for kind in ("graph", "mx4"):
            assert [r["id"] for r in db.searchMany([x[at]], {"topK": 5, "candidates": kind})[0]] == want
    db.close()
