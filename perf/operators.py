"""Measured cases of the microscaled 4-bit operators: quantisation, product, and product with top-k (scan).

A vector is held as blocks of 32 components.  A block is one scale 2^(s - 127) (s: one byte, 255 = not a number) and 32
codes of 4 bits {sign, 2 bits exponent, 1 bit mantissa}, which stand for +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}.  With m the
largest magnitude of a block, s - 127 = floor(log2 m) - 2, not below -127; a code is the nearest of the eight magnitudes to
|x| / 2^(s - 127) (ties to the even code), at most 6.  A packed row is 16 bytes for each block (component 2 i in the low half of
byte i), an even number of blocks, then one scale byte for each, filled with zeros to a multiple of 16 bytes.

  quantise  f32, bf16 or f16 rows -> packed rows, and back to the values they stand for
  product   packed queries x packed rows -> every dot product, f32
  scan      f32 queries -> packed, then the k largest dot products with packed rows for each query: ids, values, counts.
            Order: value descending, then id ascending; rows whose bit is not set in `allow` are left out.

The dimensions, batch and row counts are those of this repository's own searches: dim 384 and 512, 1000 and 4096 queries, 10 000
and 1 M rows, topK 10 (and 100 candidates for a rerank), and odd sizes around them.
"""
import torch

own = False

_DEV = "cuda"
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one query vector on its way to a scan: the latency of the call
        {"name": "quantise 1x384", "op": "quantise", "rows": 1, "dim": 384, "dtype": "f32", "pad": 0},
        # rows as an embedding model leaves them (bf16, inside a wider buffer), a dimension that ends inside a block
        {"name": "quantise 50021x1000 bf16", "op": "quantise", "rows": 50021, "dim": 1000, "dtype": "bf16", "pad": 24},
        # a whole float32 store of a million rows
        {"name": "quantise 1Mx384", "op": "quantise", "rows": 1000000, "dim": 384, "dtype": "f32", "pad": 0},
        # one query against a small collection
        {"name": "product 1x10000x384", "op": "product", "nq": 1, "rows": 10000, "dim": 384},
        # a ragged batch
        {"name": "product 37x50021x1000", "op": "product", "nq": 37, "rows": 50021, "dim": 1000},
        # a batch of the usual size, every score wanted
        {"name": "product 1000x262144x384", "op": "product", "nq": 1000, "rows": 262144, "dim": 384},
        # the largest batch
        {"name": "product 4096x65536x512", "op": "product", "nq": 4096, "rows": 65536, "dim": 512},
        # one query, small collection: latency
        {"name": "scan 1x10000x384", "op": "scan", "nq": 1, "rows": 10000, "dim": 384, "k": 10, "allow": 1.0},
        # one query over a million rows: the store is read once
        {"name": "scan 1x1Mx384", "op": "scan", "nq": 1, "rows": 1000000, "dim": 384, "k": 10, "allow": 1.0},
        # ragged sizes, a filter, and enough candidates for a rerank
        {"name": "scan 333x200003x100 k100", "op": "scan", "nq": 333, "rows": 200003, "dim": 100, "k": 100, "allow": 0.3},
        # the usual batch over a million rows
        {"name": "scan 1000x1Mx384", "op": "scan", "nq": 1000, "rows": 1000000, "dim": 384, "k": 10, "allow": 1.0},
        # the batch of the exact 8-bit scan
        {"name": "scan 4096x1Mx512", "op": "scan", "nq": 4096, "rows": 1000000, "dim": 512, "k": 10, "allow": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quantise", "product", "scan", "scan"])
    dim = 4 * _log_int(rng, 2, 256)  # the engine's dimensions are multiples of four
    if op == "quantise":
        rows = _log_int(rng, 1, 1000000)
        rows = max(1, min(rows, 384000000 // dim))
        return {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(["f32", "bf16", "f16"]), "pad": rng.choice([0, 0, 4, 7, 24])}
    nq = _log_int(rng, 1, 4096)
    if op == "product":
        rows = _log_int(rng, 64, 262144)
        rows = max(64, min(rows, 262144000 // nq))
        return {"op": op, "nq": nq, "rows": rows, "dim": dim}
    rows = _log_int(rng, 1000, 1000000)
    if dim > 512:
        rows = max(1000, rows // 2)
    return {"op": op, "nq": nq, "rows": rows, "dim": dim, "k": _log_int(rng, 1, 128), "allow": rng.choice([1.0, 1.0, 0.5, 0.02])}


# ------------------------------------------------------------------------------------------------- inputs
def _unit_rows(g, rows, dim, centres):
    """Unit vectors around centres of their own: what an embedding store holds."""
    at = torch.randint(0, centres.shape[0], (rows,), generator=g, device=_DEV)
    x = torch.randn((rows, dim), generator=g, device=_DEV)
    x += centres[at]
    x /= x.square().sum(-1, keepdim=True).sqrt_()
    return x


def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed))
    dim = case["dim"]
    centres = torch.randn((256, dim), generator=g, device=_DEV)
    if case["op"] == "quantise":
        x = _unit_rows(g, case["rows"], dim, centres).to(_DTYPES[case["dtype"]])
        if case["pad"]:  # rows inside a wider buffer
            wide = torch.zeros((case["rows"], dim + case["pad"]), dtype=x.dtype, device=_DEV)
            wide[:, :dim] = x
            x = wide[:, :dim]
        return {"op": "quantise", "dim": dim, "x": x}
    rows = _pack(_unit_rows(g, case["rows"], dim, centres))
    q = _unit_rows(g, case["nq"], dim, centres)
    if case["op"] == "product":
        return {"op": "product", "dim": dim, "q": _pack(q), "rows": rows}
    allow = None
    if case["allow"] < 1.0:  # bit i of word i / 32: row i passes the filter
        bits = torch.rand(((case["rows"] + 31) // 32, 32), generator=g, device=_DEV) < case["allow"]
        allow = (bits.to(torch.int64) << torch.arange(32, device=_DEV)).sum(-1).to(torch.int32)
    return {"op": "scan", "dim": dim, "q": q, "rows": rows, "k": case["k"], "allow": allow}


# ------------------------------------------------------------------------------------------------- plain forms
def _blocks(dim):
    return 2 * ((dim + 63) // 64)


def _pack(x):
    """Rows (any floating type) -> packed rows."""
    n, dim = x.shape
    nb = _blocks(dim)
    full = torch.zeros((n, nb * 32), dtype=torch.float32, device=x.device)
    full[:, :dim] = x
    full = full.view(n, nb, 32)
    top = full.abs().amax(-1)  # a NaN stays one
    fine = torch.isfinite(top)
    s = ((top.view(torch.int32) >> 23) - 2).clamp_(min=0)
    down = ((254 - s) << 23).view(torch.float32)  # 2^(127 - s)
    y = full * torch.where(fine, down, torch.zeros_like(down)).unsqueeze(-1)
    a = y.abs()
    code = (a > 0.25).to(torch.uint8)
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5
    code |= torch.signbit(full).to(torch.uint8) << 3
    code = torch.where(fine.unsqueeze(-1), code, torch.zeros_like(code)).view(n, nb * 16, 2)
    tail = torch.zeros((n, (nb + 15) // 16 * 16), dtype=torch.uint8, device=x.device)
    tail[:, :nb] = torch.where(fine, s, torch.full_like(s, 255))
    return torch.cat([code[..., 0] | (code[..., 1] << 4), tail], 1)


def _values(packed, dim):
    """Packed rows -> the f32 values they stand for."""
    n, nb = packed.shape[0], _blocks(dim)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float32, device=packed.device)
    step = torch.exp2(torch.arange(256, dtype=torch.float64, device=packed.device) - 127).to(torch.float32)
    step[255] = float("nan")
    byte = packed[:, : nb * 16]
    code = torch.stack([byte & 15, byte >> 4], -1).view(n, nb, 32)
    v = grid[code.to(torch.int32)] * step[packed[:, nb * 16 : nb * 17].to(torch.int32)].unsqueeze(-1)
    return v.view(n, nb * 32)[:, :dim]


def _topk(scores, k, allow):
    """The k best of each row of scores: value descending, then id ascending; ids -1 and values 0 behind the last."""
    n = scores.shape[1]
    ids = torch.arange(n, device=scores.device)
    out = torch.isnan(scores)
    if allow is not None:
        out |= ((allow[ids >> 5] >> (ids & 31)) & 1) == 0
    b = (scores + 0.0).view(torch.int32)
    b ^= (b >> 31) & 0x7FFFFFFF  # whole numbers in the order of the values
    key = b.to(torch.int64)
    key <<= 32
    key += 0xFFFFFFFF - ids
    none = torch.iinfo(torch.int64).min
    key.masked_fill_(out, none)
    best = key.topk(min(k, n), dim=1).values
    if n < k:
        best = torch.cat([best, torch.full((best.shape[0], k - n), none, device=best.device)], 1)
    got = best != none
    v = (best >> 32).to(torch.int32)
    v ^= (v >> 31) & 0x7FFFFFFF
    val = torch.where(got, v.view(torch.float32), 0.0)
    return torch.where(got, 0xFFFFFFFF - (best & 0xFFFFFFFF), -1).to(torch.int32), val, got.sum(1).to(torch.int32)


def _run_plain(state):
    dim = state["dim"]
    if state["op"] == "quantise":
        return {"values": _values(_pack(state["x"]), dim)}
    rows = _values(state["rows"], dim)
    if state["op"] == "product":
        return {"scores": _values(state["q"], dim) @ rows.T}
    scores = _values(_pack(state["q"]), dim) @ rows.T
    ids, val, count = _topk(scores, state["k"], state["allow"])
    return {"ids": ids, "values": val, "count": count}


# ------------------------------------------------------------------------------------------------- the framework's
_engines = {}


def _engine(dim):
    """The program's handle: one engine for each dimension, kept while the program runs."""
    if dim not in _engines:
        from minivectordb_amd import HipBridge
        from minivectordb_amd.pipeline import ResidentMx4

        b = HipBridge(device=torch.cuda.current_device())
        b.init(dict(dim=dim, m=16, ef=300, capacity=8, seed=1))
        _engines[dim] = ResidentMx4(b, torch.device("cuda", torch.cuda.current_device()))
    return _engines[dim]


def _run_own(state):
    mx = _engine(state["dim"])
    if state["op"] == "quantise":
        return {"values": mx.expand(mx.quantize(state["x"]))}
    if state["op"] == "product":
        return {"scores": mx.product(state["q"], state["rows"])}
    ids, val, count = mx.scan_many(mx.quantize(state["q"]), state["rows"], state["k"], state["allow"])
    return {"ids": ids, "values": val, "count": count}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------- what has to be moved
def work(case):
    dim = case["dim"]
    nb = _blocks(dim)
    packed = 16 * nb + (nb + 15) // 16 * 16
    if case["op"] == "quantise":
        size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
        return {"bytes": case["rows"] * (dim * size + packed + dim * 4), "flops": 2 * case["rows"] * dim}
    nq, rows = case["nq"], case["rows"]
    flops = 2 * nq * rows * dim
    if case["op"] == "product":
        return {"bytes": (nq + rows) * packed + 4 * nq * rows, "flops": flops}
    return {"bytes": nq * dim * 4 + rows * packed + nq * (case["k"] * 8 + 4) + (rows // 8 if case["allow"] < 1.0 else 0), "flops": flops}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _rounded64(x):
    """The values that rows stand for once quantised, from the definition: the nearest of the representable numbers."""
    n, dim = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -dim % 32)).view(n, -1, 32)
    _, e = torch.frexp(x.abs().max(-1, keepdim=True).values)  # m = f 2^e with f in [0.5, 1): floor(log2 m) = e - 1
    unit = torch.exp2((e - 3).clamp(min=-127).double())
    a = (x / unit).abs().clamp(max=6)
    # the spacing of the magnitudes is 0.5 below 2, 1 below 4, 2 above; rounding to a multiple of it is to the nearest, ties to even
    gap = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(x) * torch.round(a / gap) * gap * unit).view(n, -1)[:, :dim]


def _stands_for64(packed, dim):
    """What packed rows stand for, from the bits of a code: (-1)^sign 2^(max(exponent, 1) - 1) (1 or 0 + mantissa / 2)."""
    nb = (dim + 63) // 64 * 2
    data, s = packed[:, : 16 * nb].long(), packed[:, 16 * nb : 17 * nb].long()
    c = torch.stack((data % 16, data // 16), 2).flatten(1)
    exponent, mantissa = (c // 2) % 4, (c % 2).double()
    mag = torch.where(exponent == 0, mantissa / 2, torch.exp2(exponent.double() - 1) * (1 + mantissa / 2))
    mag = torch.where(c >= 8, -mag, mag) * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    return mag[:, :dim]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantise":
        return {"values": _rounded64(state["x"])}
    rows = _stands_for64(state["rows"], case["dim"])
    if case["op"] == "product":
        return {"scores": _stands_for64(state["q"], case["dim"]) @ rows.T}
    scores = _rounded64(state["q"]) @ rows.T
    if state["allow"] is not None:
        bit = torch.arange(32, device=scores.device)
        keep = ((state["allow"].unsqueeze(1) >> bit) & 1).bool().flatten()[: scores.shape[1]]
        scores.masked_fill_(~keep, -float("inf"))
    best = torch.topk(scores, min(case["k"], scores.shape[1]), dim=1).values
    best = torch.nn.functional.pad(best, (0, case["k"] - best.shape[1]))
    return {"ids": None, "values": torch.where(torch.isinf(best), 0.0, best), "count": None}
