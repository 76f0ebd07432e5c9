"""Microscaled 4-bit rows from their definition, in 64 bits (numpy; test infrastructure only).

The format is written down in include/mvdb_hip.h.  Nothing here is fast: rounding picks the nearest of the eight magnitudes
by its distance, products are f64 sums of the values the codes stand for, top-k is a stable sort."""
from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def blocks(dim: int) -> int:
    return 2 * ((dim + 63) // 64)


def row_bytes(dim: int) -> int:
    return 16 * blocks(dim) + (blocks(dim) + 15) // 16 * 16


def codes_and_scales(x):
    """rows (any float type, taken as 64-bit) -> (codes uint8 [n, nb, 32], scale bytes uint8 [n, nb])."""
    x = np.asarray(x, np.float64)
    n, dim = x.shape
    nb = blocks(dim)
    b = np.zeros((n, nb * 32))
    b[:, :dim] = x
    b = b.reshape(n, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 0, np.abs(np.where(np.isfinite(b), b, 0)).max(-1))
    with np.errstate(divide="ignore"):
        e = np.floor(np.log2(top))
    # floor(log2) of a value just below a power of two may round up: settle it by comparison
    ef = np.where(top > 0, e, -200).astype(np.int64)
    ef = np.where((top > 0) & (np.ldexp(1.0, ef) > top), ef - 1, ef)
    ef = np.where((top > 0) & (np.ldexp(1.0, ef + 1) <= top), ef + 1, ef)
    s = np.maximum(ef - 2, -127)
    with np.errstate(invalid="ignore"):
        y = np.abs(b) / np.ldexp(1.0, s)[..., None]
    y = np.where(bad[..., None], 0, y)
    code = np.zeros(y.shape, np.uint8)
    dist = np.abs(y - 0.0)
    for c in range(1, 8):
        d = np.abs(y - MAGNITUDES[c])
        take = (d < dist) | ((d == dist) & (c % 2 == 0))
        code = np.where(take, c, code).astype(np.uint8)
        dist = np.where(take, d, dist)
    code |= (np.signbit(b).astype(np.uint8) << 3)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    return code, np.where(bad, 255, s + 127).astype(np.uint8)


def pack(x):
    code, s = codes_and_scales(x)
    n, nb, _ = code.shape
    out = np.zeros((n, row_bytes(np.asarray(x).shape[1])), np.uint8)
    out[:, : 16 * nb] = (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(n, 16 * nb)
    out[:, 16 * nb : 17 * nb] = s
    return out


def values(packed, dim: int):
    packed = np.asarray(packed)
    n, nb = packed.shape[0], blocks(dim)
    c = packed[:, : 16 * nb]
    code = np.stack([c & 15, c >> 4], -1).reshape(n, nb, 32)
    s = packed[:, 16 * nb : 17 * nb].astype(np.int64)
    scale = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    v = np.where(code & 8, -1.0, 1.0) * MAGNITUDES[code & 7] * scale[..., None]
    return v.reshape(n, nb * 32)[:, :dim]


def products(q_packed, r_packed, dim: int):
    """(f64 sums, f64 sums of the magnitudes: what an f32 sum's error is measured by)"""
    q, r = values(q_packed, dim), values(r_packed, dim)
    with np.errstate(invalid="ignore"):
        return q @ r.T, np.abs(q) @ np.abs(r).T


def topk(scores, k: int, allow=None):
    """scores [nq, n] -> (ids, values, counts): value descending, then id ascending; NaN and rows not allowed never."""
    nq, n = scores.shape
    keep = np.ones(n, bool)
    if allow is not None:
        w = np.asarray(allow, np.uint32)
        keep = ((w[np.arange(n) >> 5] >> (np.arange(n) & 31).astype(np.uint32)) & 1).astype(bool)
    ids = np.full((nq, k), -1, np.int32)
    val = np.zeros((nq, k), np.float64)
    cnt = np.zeros(nq, np.int32)
    for i in range(nq):
        cand = np.flatnonzero(keep & ~np.isnan(scores[i]))
        order = cand[np.argsort(-(scores[i][cand] + 0.0), kind="stable")][:k]
        cnt[i] = order.size
        ids[i, : order.size] = order
        val[i, : order.size] = scores[i][order]
    return ids, val, cnt
