"""Attention over 8-bit caches (akh_attn_cached_q8, akh_attn_prefix_q8) where magnitudes are far
apart: values' scales of neighbouring keys, of keys that a row does not see and of the two sources;
queries, keys and scales near the ends of 32-bit floats.  Every tolerance is relative to what the
row's own keys add, not to the largest value that it sees."""

import numpy as np
import pytest

from test_q8 import Held, _attend, _close, _write

gpu = pytest.mark.gpu


def fine(q, held, pos, counts, scale, prefix=None, ahead=0):
    """(out, lse, their bounds) in 64 bits, head by head.

    A weight exp(x - level) is off by d: its score by (head_dim + 8) 2^-23 of its own products'
    magnitudes and, by the terms of the query, 2^-21 of them with the row's largest query in each
    one's place; the exponent of 2 by 2^-24 of itself at each of its roundings, and it lies within
    |x - top| + 2^7 of a level: 32 covers 2^7 ln 2 / 4.  The two fp16 terms of a weight leave 2^-21 of it, and of a key 2^-29 of the most that
    one adds.  Sums of n weights add n 2^-24, joins and the division a few roundings more; the
    smallest 32-bit numbers lose 2^-150 each time."""
    batch, rows, heads, hd = q.shape
    group = heads // held.shape[2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse, ltol = np.full(q.shape[:3], -np.inf), np.zeros(q.shape[:3])
    scale = float(np.float32(scale))
    for b, t, h in np.ndindex(*q.shape[:3]):
        if t >= min(int(counts[b]), rows):
            continue
        n = min(int(pos[b]) + t + 1, held.shape[1])
        k, v = held.k[b, h // group, :n], held.v[b, h // group, :n]
        if prefix is not None:
            k = np.concatenate([prefix.k[0, h // group, :ahead], k])
            v = np.concatenate([prefix.v[0, h // group, :ahead], v])
        n = len(k)
        row = q[b, t, h].astype(np.float64)
        x = k @ row * scale
        top = x.max()
        p = np.exp(x - top)
        total = p.sum()
        out[b, t, h] = p @ v / total
        lse[b, t, h] = top + np.log(total)
        d = (abs(scale) * ((hd + 8) * 2.0 ** -23 * (np.abs(k) @ np.abs(row))
                           + 2.0 ** -21 * np.abs(k).sum(1) * np.abs(row).max())
             + 2.0 ** -22 * (np.abs(x) + np.abs(x - top) + 32))
        moved, added = p * (d + 2.0 ** -21 + (n + 64) * 2.0 ** -23), np.abs(v)
        tol[b, t, h] = (moved @ added + np.abs(out[b, t, h]) * moved.sum()
                        + n * 2.0 ** -29 * (p * added.max(1)).max()) / total + 2.0 ** -140
        ltol[b, t, h] = moved.sum() / total + 2.0 ** -22 * (np.abs(x).max() + np.log(n) + 1)
    return out, lse, tol, ltol


# Blocks of 8 packed rows, of 16, of 64 and of 128, at both row sizes.
SHAPES = [(1, 8, 1, 128, 333), (3, 4, 2, 64, 333), (1, 2, 2, 64, 3000), (16, 2, 2, 64, 333),
          (6, 4, 2, 128, 333), (40, 3, 1, 64, 333), (33, 8, 2, 128, 333), (64, 4, 2, 128, 1100)]


def _cache(pkg, be, k, v):
    batch, n, kvh, hd = k.shape
    held = Held(batch, n, kvh, hd)
    cache = pkg.hip.Q8Cache(be, batch, n, kvh, hd)
    _write(pkg, be, cache, k, v, [0] * batch, None)
    held.write(k, v, [0] * batch, [n] * batch)
    return cache, held


def _biased(rng, batch, n, kvh, hd, bias, scale):
    """K rows whose scores with rows of _queries have bias [batch, n] on top."""
    k = rng.standard_normal((batch, n, kvh, hd))
    k[..., 0] = np.broadcast_to(bias, (batch, n))[..., None] / scale
    return k


def _queries(rng, *shape):
    q = rng.standard_normal(shape)
    q[..., 0] = 1
    return q.astype(np.float32)


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,n", SHAPES)
def test_values_of_any_scale(backend, pkg, rows, heads, kvh, hd, n):
    rng = np.random.default_rng(rows * heads + hd + n)
    batch, scale = 7, 0.125
    last = n - rows  # rows from here on are not for all to see
    bias, size = np.zeros((batch, n)), np.zeros((batch, n))
    odd = rng.integers(0, min(32, last), batch)  # of the first keys: levels start at them
    for b, (live, other) in enumerate([(0, 126), (-110, 0), (0, 118), (-122, 0), (100, 0)]):
        size[b] = live + rng.integers(-3, 4, n)
        size[b, odd[b]] = other  # one key, which weighs nothing
        bias[b, odd[b]] = -200
    size[5, n - 1] = 126  # the last row's own key
    size[6] = rng.integers(-45, 46, n)  # every key adds about the same
    bias[6] = -np.log(2) * size[6]
    k = _biased(rng, batch, n, kvh, hd, bias, scale).astype(np.float32)
    v = np.clip(rng.standard_normal(k.shape), -1.9, 1.9) * np.exp2(size)[..., None, None]
    cache, held = _cache(pkg, backend, k, v.astype(np.float32))
    q = _queries(rng, batch, rows, heads, hd)
    pos = [last] * batch
    got, lse = _attend(pkg, backend, q, cache, pos, None, scale)
    want, wl, tol, lt = fine(q, held, pos, [rows] * batch, scale)
    _close(got, want, tol)
    _close(lse, wl, lt)
    behind = pos[0] + np.arange(rows) < n - 1
    assert np.abs(got[5, behind]).max(initial=0) < 100  # (the others' sums are small)


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,n", SHAPES)
@pytest.mark.parametrize("size", [40, -100, 100])
def test_scores_of_2_to_the_30(backend, pkg, rows, heads, kvh, hd, n, size):
    # Scores 10^7 apart: one key takes all, and a level next to 2^30 is a multiple of 64 and
    # more in 32 bits.
    rng = np.random.default_rng(rows * heads + hd)
    k = np.zeros((1, n, kvh, hd), np.float32)
    v = (rng.standard_normal(k.shape) * 2.0 ** size).astype(np.float32)
    at = int(rng.integers(n - rows))
    k[0, :, :, 0] = 2.0 ** 30
    k[0, at, :, 0] = 2.0 ** 30 + 2.0 ** 24
    cache, held = _cache(pkg, backend, k, v)
    q = np.zeros((1, rows, heads, hd), np.float32)
    q[..., 0] = 1
    got, lse = _attend(pkg, backend, q, cache, [n - rows], None, 1.0)
    want = held.v[0, np.arange(heads) // (heads // kvh), at]
    # A weight of one: its two terms, the sum's reciprocal and products with it, in 32 bits.
    _close(got[0], np.broadcast_to(want, got[0].shape), np.abs(want) * 2.0 ** -19)
    _close(lse[0], np.full((rows, heads), held.k[0, 0, at, 0]), 2.0 ** 30 * 2.0 ** -21)


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,n", SHAPES)
@pytest.mark.parametrize("own,pre", [(58, -100), (-100, 58), (85, -85), (-85, 85), (115, -115),
                                     (-120, 0), (0, 119)])
def test_parts_whose_values_are_far_apart(backend, pkg, rows, heads, kvh, hd, n, own, pre):
    # Own rows and prefix weigh the same, and one key of either, which weighs nothing, has a
    # scale of its own.
    rng = np.random.default_rng(rows * heads + hd + 200 + own)
    batch, scale, ahead, most = 2, 0.125, 200, min(n, 333)
    parts = []
    for slots, length, exp in ((batch, most, own), (1, ahead, pre)):
        bias, size = np.zeros((slots, length)), np.full((slots, length), float(exp))
        bias[:, 5], size[:, 5] = -200, -10
        k = _biased(rng, slots, length, kvh, hd, bias, scale).astype(np.float32)
        v = rng.standard_normal(k.shape) * np.exp2(size)[..., None, None]
        parts.append(_cache(pkg, backend, k, v.astype(np.float32)))
    (cache, held), (prefix, pheld) = parts
    q = _queries(rng, batch, rows, heads, hd)
    pos = [most - rows, most - rows - 40]
    got, lse = _attend(pkg, backend, q, cache, pos, None, scale, prefix, ahead)
    want, wl, tol, lt = fine(q, held, pos, [rows] * batch, scale, pheld, ahead)
    _close(got, want, tol)
    _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,n", SHAPES)
@pytest.mark.parametrize("most", [70, 85, 115])
def test_values_that_grow_along_the_keys(backend, pkg, rows, heads, kvh, hd, n, most):
    # Waves, halves and splits of the keys meet scales of their own; growing and falling.
    rng = np.random.default_rng(rows * heads + hd + n + most)
    batch, scale = 2, 0.125
    size = np.linspace(-most, most, n)
    k = _biased(rng, batch, n, kvh, hd, 0, scale).astype(np.float32)
    v = rng.standard_normal(k.shape) * np.exp2(np.stack([size, size[::-1]]))[..., None, None]
    cache, held = _cache(pkg, backend, k, v.astype(np.float32))
    q = _queries(rng, batch, rows, heads, hd)
    pos = [n - rows, n - rows - 40]
    got, lse = _attend(pkg, backend, q, cache, pos, None, scale)
    want, wl, tol, lt = fine(q, held, pos, [rows] * batch, scale)
    _close(got, want, tol)
    _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,n", SHAPES)
def test_queries_of_any_scale(backend, pkg, rows, heads, kvh, hd, n):
    # q and K scaled against each other, from subnormal queries to those next to 2^127; among a
    # sequence's rows some of ordinary scores and some of none.
    rng = np.random.default_rng(rows * heads + hd + n)
    by = [-104, -107, -114, -118, -124, 60, 100, 117]
    batch, n, scale = len(by), min(n, 333), 0.125
    k = rng.standard_normal((batch, n, kvh, hd)) * np.exp2(-np.float64(by))[:, None, None, None]
    v = rng.standard_normal(k.shape)
    q = rng.standard_normal((batch, rows, heads, hd)) * np.exp2(np.float64(by))[:, None, None, None]
    q[:5, 1::3] *= 2.0 ** -20
    with np.errstate(under="ignore"):
        k, v, q = (x.astype(np.float32) for x in (k, v, q))
    cache, held = _cache(pkg, backend, k, v)
    pos = [n - rows] * batch
    got, lse = _attend(pkg, backend, q, cache, pos, None, scale)
    want, wl, tol, lt = fine(q, held, pos, [rows] * batch, scale)
    _close(got, want, tol)
    _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,n", SHAPES)
@pytest.mark.parametrize("scale,by_q,by_k", [(2.0 ** 127, -120, -10), (3e38, -60, -70),
                                             (2.0 ** 100, -126, 20), (2.0 ** -140, 60, 78),
                                             (2.0 ** -126, 120, 4), (-2.0 ** 90, 30, -122),
                                             (0.0, 0, 0)])
def test_any_scale(backend, pkg, rows, heads, kvh, hd, n, scale, by_q, by_k):
    rng = np.random.default_rng(rows * heads + hd + n)
    batch, n = 2, min(n, 333)
    scale = float(np.float32(scale))
    k = (rng.standard_normal((batch, n, kvh, hd)) * 2.0 ** by_k).astype(np.float32)
    v = rng.standard_normal(k.shape).astype(np.float32)
    q = (rng.standard_normal((batch, rows, heads, hd)) * 2.0 ** by_q).astype(np.float32)
    cache, held = _cache(pkg, backend, k, v)
    pos = [n - rows, n - rows - 70]
    got, lse = _attend(pkg, backend, q, cache, pos, None, scale)
    want, wl, tol, lt = fine(q, held, pos, [rows] * batch, scale)
    _close(got, want, tol)
    _close(lse, wl, lt)
