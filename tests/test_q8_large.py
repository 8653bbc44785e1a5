"""Attention over 8-bit caches larger than the machine's own caches, whose codes are read past them
unless several groups of query rows share them: the blocks of 8 packed rows with two waves and
those of 16 rows, at both row sizes, with one split of the keys and with several, against 64 bits."""

import numpy as np
import pytest

from test_q8 import Held, _attend, _close, _rows, _write, attention

gpu = pytest.mark.gpu


def _same_slots(pkg, be, rng, slots, most, kvh, hd):
    """A cache whose slots all hold the same rows, and what one of them holds."""
    held = Held(1, most, kvh, hd)
    k, v = (_rows(rng, 1, most, kvh, hd, 1) for _ in range(2))
    held.write(k, v, [0], [most])
    size = pkg.hip.q8_cache_bytes(1, most, kvh, hd)
    one = be.zeros(size, np.uint8)
    _write(pkg, be, pkg.hip.Q8Cache(be, 1, most, kvh, hd, data=one), k, v, [0], None)
    heads = size // (2 * (1 + (64 if hd <= 64 else 128)))
    parts = np.split(one.download(np.uint8), [size // 2 - heads, size - 2 * heads, size - heads])
    data = be.tensor(np.concatenate([np.tile(p, slots) for p in parts]))
    return pkg.hip.Q8Cache(be, slots, most, kvh, hd, data=data), held


@gpu
@pytest.mark.parametrize("batch,rows,heads,kvh,hd,most", [
    (64, 1, 16, 16, 128, 400), (24, 1, 8, 8, 128, 3100),   # 8 rows, two waves
    (64, 1, 13, 13, 64, 1024), (24, 1, 12, 12, 50, 3100),
    (64, 16, 8, 8, 128, 800), (12, 12, 4, 4, 100, 9000),   # 16 rows
    (64, 10, 8, 8, 64, 1700), (12, 9, 8, 8, 64, 9000),
    (64, 5, 16, 4, 128, 2048), (12, 5, 16, 4, 128, 9000),  # in two groups
    (64, 3, 16, 4, 64, 3200)])
def test_codes_past_the_caches(backend, pkg, batch, rows, heads, kvh, hd, most):
    rng = np.random.default_rng(batch + rows + most)
    assert batch * kvh * most * 2 * (64 if hd <= 64 else 128) > 96 << 20
    cache, held = _same_slots(pkg, backend, rng, batch, most, kvh, hd)
    lens = [max(rows, most - 37 * b * (b % 5)) for b in range(batch)]
    counts = [max(0, rows - b % 3) if rows > 1 else 1 - (b % 7 == 6) for b in range(batch)]
    pos = [n - c for n, c in zip(lens, counts)]
    q = rng.standard_normal((batch, rows, heads, hd)).astype(np.float32)
    got, lse = _attend(pkg, backend, q, cache, pos, counts, hd ** -0.5)
    for b in {0, 1, 4, 6, batch // 2, batch - 1}:
        pick = {(0, t, h) for t in {0, rows // 2, rows - 1} for h in {0, heads // 2, heads - 1}}
        want, wl, tol, lt = attention(q[b:b + 1], held, pos[b:b + 1], counts[b:b + 1], hd ** -0.5,
                                      pick=pick)
        at = tuple(np.array(sorted(pick)).T)
        _close(got[b:b + 1][at], want[at], tol[at])
        _close(lse[b:b + 1][at], wl[at], lt[at])
    behind = np.arange(rows) >= np.array(counts)[:, None]
    assert (got[behind] == 0).all() and np.isneginf(lse[behind]).all()
    assert np.isfinite(got).all() and np.isfinite(lse[~behind]).all()
