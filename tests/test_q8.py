"""8-bit caches (akh_cache_write_q8, akh_cache_read_q8) and the attention that
reads them (akh_attn_cached_q8, akh_attn_prefix_q8), against their definitions
in 64 bits.

Quantised values are compared for equality: the scale is a power of two, so
there is one rounding and no room for another result.  Attention's bound is
derived per case in ``_bounds``.
"""

import ctypes as C

import numpy as np
import pytest

gpu = pytest.mark.gpu


# ---- definitions in 64 bits ----------------------------------------------


def quantise(x):
    """Values that rows x [..., head_dim] (float32) have in the cache."""
    x = x.astype(np.float64)
    top = np.abs(x).max(-1)
    with np.errstate(all="ignore"):
        m, k = np.frexp(np.where(np.isfinite(top), top, 0.0))
        e = np.maximum(-126, k - 7 + (m > 127 / 128))
        step = np.ldexp(1.0, e)[..., None]
        code = np.rint(x / step)
        # 64 * 2^122 is no 32-bit number: the code below it.
        out = np.where(e[..., None] == 122, np.clip(code, -63, 63), code) * step
    out[~np.isfinite(top)] = np.nan
    return out


class Held:
    """What a cache [slots, kv_heads, max_rows, head_dim] holds."""

    def __init__(self, slots, max_rows, kv_heads, head_dim):
        self.shape = (slots, max_rows, kv_heads, head_dim)
        self.k = np.zeros((slots, kv_heads, max_rows, head_dim))
        self.v = np.zeros_like(self.k)

    def write(self, k, v, pos, counts):
        """k, v: float32 [batch, rows, kv_heads, head_dim]."""
        for which, x in ((self.k, k), (self.v, v)):
            q = quantise(x)
            for b in range(x.shape[0]):
                for t in range(min(int(counts[b]), x.shape[1])):
                    if int(pos[b]) + t < self.shape[1]:
                        which[b, :, int(pos[b]) + t] = q[b, t]


def attention(q, held, pos, counts, scale, prefix=None, prefix_len=0, pick=None):
    """(out, lse, out bound, lse bound) of q float32 [batch, rows, heads, hd];
    pick: of these (b, t, h) only."""
    batch, rows, heads, hd = q.shape
    group = heads // held.shape[2]
    out = np.zeros(q.shape)
    lse = np.full(q.shape[:3], -np.inf)
    otol, ltol = np.zeros(q.shape), np.zeros(q.shape[:3])
    for b in range(batch):
        for t in range(min(int(counts[b]), rows)):
            n = min(int(pos[b]) + t + 1, held.shape[1])
            for h in range(heads):
                if pick is not None and (b, t, h) not in pick:
                    continue
                k, v = held.k[b, h // group, :n], held.v[b, h // group, :n]
                if prefix is not None:
                    m = min(prefix_len, prefix.shape[1])
                    k = np.concatenate([prefix.k[0, h // group, :m], k])
                    v = np.concatenate([prefix.v[0, h // group, :m], v])
                with np.errstate(all="ignore"):
                    x = (k @ q[b, t, h].astype(np.float64)) * float(np.float32(scale))
                    top = x.max()
                    p = np.exp(x - top)
                    out[b, t, h] = p @ v / p.sum()
                    lse[b, t, h] = top + np.log(p.sum())
                    a, l = _bounds(q[b, t, h], k, v, x, scale)
                otol[b, t, h], ltol[b, t, h] = a, l
    return out, lse, otol, ltol


def _bounds(q, k, v, x, scale):
    """A score is a sum of head_dim products in f32 of q, whose two fp16 terms
    leave 2^-22 of its row's largest magnitude, and exact codes, times a
    scale that is rounded twice more: at most (head_dim + 8) 2^-23 of the sum
    of magnitudes off (the row's largest in q's place).  e^x moves by as much, and by 2^-22 of its
    argument and its own rounding: the argument is x - max in units of ln 2,
    rounded to 2^-24 of it.  Sums over n weights add at most n 2^-24, the two
    terms of a weight 2^-22, joins and the division a few roundings more."""
    n, hd = k.shape
    worst = np.abs(k).sum(1).max() * np.abs(q.astype(np.float64)).max() * abs(scale)
    score = (hd + 8) * 2.0 ** -23 * worst
    weight = score + 2.0 ** -22 * (np.abs(x).max() + 4)
    total = 2 * weight + (n + 64) * 2.0 ** -23
    return total * np.abs(v).max() + 1e-38, total + 2.0 ** -22 * (np.abs(x).max() + np.log(n) + 1)


# ---- device side -----------------------------------------------------------


def _u32(be, a):
    return be.tensor(np.asarray(a, np.uint32))


def _write(pkg, be, cache, k, v, pos, counts, stride=None):
    batch, rows, kvh, hd = k.shape
    stride = stride or kvh * hd
    bufs = []
    for x in (k, v):
        wide = np.full((batch * rows, stride), 7.5, np.float32)
        wide[:, :kvh * hd] = x.reshape(batch * rows, -1)
        bufs.append(be.tensor(wide))
    be.cache_write_q8(*bufs, cache, batch, rows, stride, _u32(be, pos),
                      None if counts is None else _u32(be, counts))


def _read(be, cache, batch, rows, pos, counts, stride=None):
    kvh, hd = cache.c.kv_heads, cache.c.head_dim
    stride = stride or kvh * hd
    out = [be.tensor(np.full((batch * rows, stride), 3.25, np.float32)) for _ in range(2)]
    be.cache_read_q8(cache, *out, batch, rows, stride, _u32(be, pos),
                     None if counts is None else _u32(be, counts))
    got = [o.download().reshape(batch * rows, stride) for o in out]
    for g in got:
        assert (g[:, kvh * hd:] == 3.25).all()
    return [g[:, :kvh * hd].reshape(batch, rows, kvh, hd) for g in got]


def _attend(pkg, be, q, cache, pos, counts, scale, prefix=None, prefix_len=0, max_len=0,
            stride=None, want_lse=True):
    h = pkg.hip
    batch, rows, heads, hd = q.shape
    stride = stride or heads * hd
    wide = np.full((batch * rows, stride), 11.0, np.float32)
    wide[:, :heads * hd] = q.reshape(batch * rows, -1)
    dq, do = be.tensor(wide), be.tensor(np.full((batch * rows, stride), 3.25, np.float32))
    lse = be.tensor(np.full(batch * rows * heads, 3.25, np.float32)) if want_lse else None
    shape = h.AttnQ8(batch, rows, heads, stride, stride, scale, max_len)
    size = h.attn_q8_workspace(shape, cache, prefix)
    ws = be.tensor(np.full(size + 4, 0xFF, np.uint8))  # NaN: its contents need no preparation
    dp, dc = _u32(be, pos), None if counts is None else _u32(be, counts)
    if prefix is None:
        be.attn_cached_q8(dq, cache, do, lse, shape, dp, dc, ws, size)
    else:
        be.attn_prefix_q8(dq, prefix, _u32(be, [prefix_len]), cache, do, lse, shape, dp, dc, ws,
                          size)
    got = do.download().reshape(batch * rows, stride)
    assert (got[:, heads * hd:] == 3.25).all()
    return (got[:, :heads * hd].reshape(q.shape),
            lse.download().reshape(q.shape[:3]) if want_lse else None)


def _close(got, want, tol):
    with np.errstate(invalid="ignore"):
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        bad = ~same & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4],
                           np.broadcast_to(tol, got.shape)[bad][:4])


def _rows(rng, batch, rows, kvh, hd, spread=4):
    """Rows of magnitudes 2^-spread .. 2^spread."""
    x = rng.standard_normal((batch, rows, kvh, hd))
    return (x * np.exp2(rng.uniform(-spread, spread, (batch, rows, kvh, 1)))).astype(np.float32)


def _filled(pkg, be, rng, slots, max_rows, kvh, hd, stale=True, spread=2):
    """A cache whose rows are all written, and what it holds; `stale`: rows
    that the caller's lengths leave out are to be written over by _poison."""
    held = Held(slots, max_rows, kvh, hd)
    cache = pkg.hip.Q8Cache(be, slots, max_rows, kvh, hd)
    k, v = (_rows(rng, slots, max_rows, kvh, hd, spread) for _ in range(2))
    pos, counts = np.zeros(slots), np.full(slots, max_rows)
    _write(pkg, be, cache, k, v, pos, counts)
    held.write(k, v, pos, counts)
    return cache, held


def _poison(pkg, be, cache, lens):
    """NaN rows behind each slot's first lens[b]: an attention that reads them
    shows it."""
    slots, most = cache.c.slots, cache.c.max_rows
    bad = np.full((slots, most, cache.c.kv_heads, cache.c.head_dim), np.nan, np.float32)
    _write(pkg, be, cache, bad, bad, lens, np.maximum(0, most - np.asarray(lens)))


# ---- the cache ---------------------------------------------------------------


def test_quantise_is_within_half_a_step():
    rng = np.random.default_rng(0)
    x = _rows(rng, 7, 5, 3, 64, 30)
    off = np.abs(quantise(x) - x)
    top = np.abs(x).max(-1, keepdims=True)
    assert (off <= top / 127 + 2.0 ** -127).all()
    # 127 steps are the row's largest magnitude or more, and the half of them not.
    assert np.array_equal(quantise(np.float32([[127.0, 1.0]])), [[127.0, 1.0]])
    assert np.array_equal(quantise(np.float32([[127.5, 1.0]])), [[128.0, 2.0 * np.rint(0.5)]])
    assert np.array_equal(quantise(np.float32([[0.0, 0.0]])), [[0.0, 0.0]])


def test_cache_bytes(pkg):
    h = pkg.hip
    assert h.q8_cache_bytes(2, 33, 3, 64) == 2 * 2 * 3 * 64 * 65
    assert h.q8_cache_bytes(1, 1, 1, 1) == 2 * 32 * 65
    assert h.q8_cache_bytes(5, 64, 2, 65) == 2 * 5 * 2 * 64 * 129
    assert h.q8_cache_bytes(4, 1 << 20, 8, 128) == 2 * (4 << 20) * 8 * 129  # past 32 bits
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (1, 1, 1, 129),
                (1, (1 << 30) + 1, 1, 1), (1 << 31, 1 << 30, 1 << 31, 128)):
        with pytest.raises(h.InvalidArgument):
            h.q8_cache_bytes(*bad)


SHAPES = [(4, 64), (1, 128), (3, 33), (2, 1), (5, 80), (7, 4), (2, 127)]


@gpu
@pytest.mark.parametrize("kvh,hd", SHAPES)
@pytest.mark.parametrize("wide", [0, 5, 8])
def test_rows_round_trip(backend, pkg, kvh, hd, wide):
    rng = np.random.default_rng(kvh * 1000 + hd + wide)
    slots, most, batch, rows = 6, 45, 5, 7
    cache, held = _filled(pkg, backend, rng, slots, most, kvh, hd, spread=20)
    k, v = (_rows(rng, batch, rows, kvh, hd, 20) for _ in range(2))
    pos, counts = [0, 3, 44, 38, 45], [7, 0, 5, 100, 2]  # past the end, none, more than rows
    _write(pkg, backend, cache, k, v, pos, counts, kvh * hd + wide)
    held.write(k, v, pos, counts)
    # Everything, the rows that were not the step's included.
    got = _read(backend, cache, slots, most, [0] * slots, None, kvh * hd + wide)
    assert np.array_equal(got[0], held.k.transpose(0, 2, 1, 3))
    assert np.array_equal(got[1], held.v.transpose(0, 2, 1, 3))
    # A step's rows; what is not the step's reads zero.
    got = _read(backend, cache, batch, rows, pos, counts, kvh * hd + wide)
    for which, x in zip((held.k, held.v), got):
        for b in range(batch):
            for t in range(rows):
                live = t < counts[b] and pos[b] + t < most
                assert np.array_equal(x[b, t], which[b, :, pos[b] + t] if live else
                                      np.zeros((kvh, hd)))


@gpu
@pytest.mark.parametrize("hd", [64, 100])
def test_rows_at_the_edges(backend, pkg, hd):
    # Largest and least magnitudes, a power of two and its neighbours, zeros,
    # ties, subnormals, NaN and infinities.
    big = np.finfo(np.float32).max
    tops = [big, 127.0, 127.5, np.nextafter(np.float32(127), np.float32(128)), 128.0, 1.0, 2.0 ** -119,
            2.0 ** -120, 2.0 ** -126, 2.0 ** -127, 2.0 ** -149, 0.0, 126.5, 63.5, 63.75, np.nan,
            np.inf, -np.inf]
    n = len(tops)
    rng = np.random.default_rng(hd)
    x = (rng.uniform(-1, 1, (1, n, 1, hd)) * np.float64(1)).astype(np.float32)
    with np.errstate(all="ignore"):
        x = (x * np.array(tops, np.float32).reshape(1, n, 1, 1)).astype(np.float32)
    x[0, 1, 0, 1:9] = [0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5, 125.5]
    x[0, :, 0, 0] = tops
    for i in (15, 16, 17):
        x[0, i, 0, 1:] = rng.standard_normal(hd - 1)
    v = -x[:, ::-1]
    cache = pkg.hip.Q8Cache(backend, 1, n, 1, hd)
    _write(pkg, backend, cache, x, np.ascontiguousarray(v), [0], None)
    gk, gv = _read(backend, cache, 1, n, [0], None)
    assert np.array_equal(gk, quantise(x), equal_nan=True)
    assert np.array_equal(gv, quantise(v), equal_nan=True)
    assert np.isnan(gk[0, 15:]).all() and not np.isnan(gk[0, :15]).any()


@gpu
def test_read_one_side_and_from_a_fused_projection(backend, pkg):
    rng = np.random.default_rng(5)
    batch, rows, heads, kvh, hd = 3, 4, 6, 2, 64
    width = (heads + 2 * kvh) * hd
    qkv = rng.standard_normal((batch * rows, width)).astype(np.float32)
    buf = backend.tensor(qkv)
    cache = pkg.hip.Q8Cache(backend, batch, 10, kvh, hd)
    pos = _u32(backend, [0, 2, 6])
    backend.cache_write_q8(buf.offset(4 * heads * hd), buf.offset(4 * (heads + kvh) * hd), cache,
                           batch, rows, width, pos)
    want = quantise(qkv.reshape(batch, rows, heads + 2 * kvh, hd))
    out = backend.zeros(batch * rows * kvh * hd)
    backend.cache_read_q8(cache, out, None, batch, rows, kvh * hd, pos)
    assert np.array_equal(out.download().reshape(batch, rows, kvh, hd), want[:, :, heads:heads + kvh])
    backend.cache_read_q8(cache, None, out, batch, rows, kvh * hd, pos)
    assert np.array_equal(out.download().reshape(batch, rows, kvh, hd), want[:, :, heads + kvh:])


# ---- attention ----------------------------------------------------------------


@gpu
@pytest.mark.parametrize("heads,kvh,hd", [(4, 4, 64), (2, 2, 128), (6, 2, 64), (8, 1, 128),
                                          (3, 3, 33), (2, 2, 1), (4, 2, 80), (12, 1, 16)])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 17, 40])
def test_attention_over_the_cache(backend, pkg, heads, kvh, hd, rows):
    rng = np.random.default_rng(heads * 100 + hd + rows)
    lens = [rows, rows + 31, 64 + rows, 33 + rows, 200 + rows, 1 + rows]
    slots, most = len(lens), max(lens) + 3
    counts = [rows, rows, max(0, rows - 2), 0, rows + 5, 1]
    pos = [n - min(c, rows) for n, c in zip(lens, counts)]
    cache, held = _filled(pkg, backend, rng, slots, most, kvh, hd)
    _poison(pkg, backend, cache, lens)
    q = rng.standard_normal((slots, rows, heads, hd)).astype(np.float32)
    scale = hd ** -0.5
    got, lse = _attend(pkg, backend, q, cache, pos, counts, scale, stride=heads * hd + 3)
    want, wl, tol, lt = attention(q, held, pos, counts, scale)
    assert (got[np.arange(rows) >= np.array(counts)[:, None]] == 0).all()
    _close(got, want, tol)
    _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("heads,kvh,hd,batch,length,max_len", [
    (2, 2, 64, 1, 1, 0), (2, 2, 64, 1, 5000, 0), (1, 1, 128, 2, 3001, 0), (4, 1, 64, 3, 2500, 64),
    (2, 1, 128, 1, 4097, 9000), (5, 5, 64, 40, 130, 0), (3, 1, 40, 2, 2049, 0),
])
def test_attention_over_long_rows(backend, pkg, heads, kvh, hd, batch, length, max_len):
    # One axis long enough to be split, sequences of uneven lengths, and a
    # launch shaped for shorter or longer ones than there are.
    rng = np.random.default_rng(length + heads)
    lens = [max(1, length - 37 * i * i) for i in range(batch)]
    cache, held = _filled(pkg, backend, rng, batch, length, kvh, hd)
    _poison(pkg, backend, cache, lens)
    for rows in (1, 2):
        q = rng.standard_normal((batch, rows, heads, hd)).astype(np.float32)
        pos = [max(0, n - rows) for n in lens]
        counts = [min(rows, n) for n in lens]
        got, lse = _attend(pkg, backend, q, cache, pos, counts, 0.125, max_len=max_len)
        want, wl, tol, lt = attention(q, held, pos, counts, 0.125)
        _close(got, want, tol)
        _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("heads,kvh,hd,batch,rows", [(4, 4, 64, 3, 1), (4, 2, 128, 5, 4),
                                                     (2, 2, 64, 37, 1), (6, 1, 80, 6, 3),
                                                     (2, 2, 64, 64, 2), (3, 3, 128, 17, 1)])
@pytest.mark.parametrize("most,ahead", [(1, 1), (31, 0), (64, 40), (700, 700), (2100, 1999),
                                        (96, 5000)])
def test_attention_behind_a_prefix(backend, pkg, heads, kvh, hd, batch, rows, most, ahead):
    rng = np.random.default_rng(heads + hd + batch + most)
    prefix, pheld = _filled(pkg, backend, rng, 2, most, kvh, hd)  # slot 0 is the one
    _poison(pkg, backend, prefix, [min(ahead, most), 0])
    lens = [rows + (i * 17) % 90 for i in range(batch)]
    counts = [rows - (i % (rows + 1)) if rows > 1 else 1 - (i % 5 == 3) for i in range(batch)]
    pos = [n - c for n, c in zip(lens, counts)]
    cache, held = _filled(pkg, backend, rng, batch + 1, max(lens), kvh, hd)
    _poison(pkg, backend, cache, lens + [0])
    q = rng.standard_normal((batch, rows, heads, hd)).astype(np.float32)
    scale = hd ** -0.5
    got, lse = _attend(pkg, backend, q, cache, pos, counts, scale, prefix, ahead)
    want, wl, tol, lt = attention(q, held, pos, counts, scale, pheld, ahead)
    _close(got, want, tol)
    _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_uneven_magnitudes(backend, pkg, hd):
    # Scores far apart (one key takes all, the others underflow), a flat row, K and V rows whose
    # scales are far apart, large and tiny values throughout.
    rng = np.random.default_rng(hd)
    batch, n = 5, 300
    k, v = (rng.standard_normal((batch, n, 1, hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((batch, 1, 1, hd)).astype(np.float32)
    k[0] *= 40
    k[1] = 0
    v[2] *= np.exp2(rng.integers(-20, 20, (n, 1, 1))).astype(np.float32)
    k[2] *= np.exp2(rng.integers(-12, 1, (n, 1, 1))).astype(np.float32)
    k[3] *= np.float32(1e25)
    q[3] *= np.float32(1e-25)
    v[3] *= np.float32(1e30)
    k[4] *= np.float32(1e-25)
    q[4] *= np.float32(1e25)
    v[4] *= np.float32(1e-30)
    held = Held(batch, n, 1, hd)
    cache = pkg.hip.Q8Cache(backend, batch, n, 1, hd)
    pos = np.zeros(batch)
    _write(pkg, backend, cache, k, v, pos, None)
    held.write(k, v, pos, [n] * batch)
    last = [n - 1] * batch
    got, lse = _attend(pkg, backend, q, cache, last, None, 0.3)
    want, wl, tol, lt = attention(q, held, last, [1] * batch, 0.3)
    _close(got, want, tol)
    _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd", [(1, 8, 1, 128), (5, 4, 2, 64), (16, 2, 1, 64),
                                               (24, 2, 1, 100), (40, 3, 1, 64), (33, 8, 2, 128)])
def test_attention_of_uneven_rows(backend, pkg, rows, heads, kvh, hd):
    # The same in every tile of rows: levels that rise along the keys, values'
    # scales far from 1 in one head, K's beyond 2^90 in another sequence.
    rng = np.random.default_rng(rows * heads)
    batch, n, ahead = 3, 333, 150
    k, v = (rng.standard_normal((batch, n, kvh, hd)) for _ in range(2))
    q = rng.standard_normal((batch, rows, heads, hd))
    k[0] *= np.linspace(0, 30, n)[:, None, None]      # ever larger scores
    v[0] *= np.exp2(rng.integers(-30, 30, (n, 1, 1)))
    k[1], q[1] = k[1] * 2.0 ** 100, q[1] * 2.0 ** -100
    v[1, :, 0] *= 2.0 ** np.linspace(-70, 70, n)[:, None]
    v[2, n // 2:] *= 2.0 ** 90
    k, v, q = (x.astype(np.float32) for x in (k, v, q))
    held = Held(batch, n, kvh, hd)
    cache = pkg.hip.Q8Cache(backend, batch, n, kvh, hd)
    _write(pkg, backend, cache, k, v, [0] * batch, None)
    held.write(k, v, [0] * batch, [n] * batch)
    prefix, pheld = _filled(pkg, backend, rng, 1, ahead, kvh, hd)
    pos = [n - rows, n - rows - 60, n - rows - 1]
    for pre, ph, some in ((None, None, 0), (prefix, pheld, ahead)):
        got, lse = _attend(pkg, backend, q, cache, pos, None, 0.2, pre, some)
        want, wl, tol, lt = attention(q, held, pos, [rows] * batch, 0.2, ph, some)
        _close(got, want, tol)
        _close(lse, wl, lt)


@gpu
@pytest.mark.parametrize("batch,rows,heads,kvh,hd,length,ahead", [
    (4, 16, 32, 4, 100, 4000, 0), (2, 128, 8, 8, 50, 8000, 0), (16, 33, 8, 8, 80, 3500, 0),
    (32, 64, 16, 16, 128, 500, 0), (32, 128, 8, 8, 64, 700, 0), (64, 33, 16, 16, 64, 400, 0),
    (40, 1, 16, 16, 128, 3, 20000), (64, 2, 16, 16, 128, 3, 8200), (64, 4, 16, 4, 64, 40, 8200),
    (20, 40, 16, 16, 128, 200, 4000), (20, 24, 16, 4, 64, 100, 4000),
    (60, 1, 32, 32, 64, 2, 16000)])
def test_attention_of_many_rows(backend, pkg, batch, rows, heads, kvh, hd, length, ahead):
    # Enough rows and keys for blocks of 64 and 128 rows, with one split and
    # with several; a sample of the rows against 64 bits.
    rng = np.random.default_rng(batch + rows + length)
    lens = [max(1, length - 13 * i) for i in range(batch)]
    counts = [min(n, max(0, rows - 5 * (i % 4)) if rows > 4 else rows - i % (rows + 1))
              for i, n in enumerate(lens)]
    pos = [n - c for n, c in zip(lens, counts)]
    cache, held = _filled(pkg, backend, rng, batch, length, kvh, hd)
    _poison(pkg, backend, cache, lens)
    prefix = pheld = None
    if ahead:
        prefix, pheld = _filled(pkg, backend, rng, 1, ahead + 30, kvh, hd)
        _poison(pkg, backend, prefix, [ahead])
    q = rng.standard_normal((batch, rows, heads, hd)).astype(np.float32)
    got, lse = _attend(pkg, backend, q, cache, pos, counts, hd ** -0.5, prefix, ahead)
    pick = {(int(rng.integers(batch)), int(rng.integers(rows)), int(rng.integers(heads)))
            for _ in range(150)}
    pick |= {(b, max(0, counts[b] - 1), heads - 1) for b in range(batch)}
    want, wl, tol, lt = attention(q, held, pos, counts, hd ** -0.5, pheld, ahead, pick)
    at = tuple(np.array(sorted(pick)).T)
    _close(got[at], want[at], tol[at])
    _close(lse[at], wl[at], lt[at])
    behind = np.arange(rows) >= np.array(counts)[:, None]
    assert (got[behind] == 0).all() and np.isneginf(lse[behind]).all()
    assert np.isfinite(got).all() and np.isfinite(lse[~behind]).all()


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,batch", [(700, 4, 2, 64, 2), (515, 16, 16, 128, 4),
                                                     (1029, 32, 8, 112, 2)])
def test_attention_of_a_whole_prompt(backend, pkg, rows, heads, kvh, hd, batch):
    # Every row sees one key more than the row before it, from the first.
    rng = np.random.default_rng(rows)
    cache, held = _filled(pkg, backend, rng, batch, rows + 40, kvh, hd)
    prefix, pheld = _filled(pkg, backend, rng, 1, 70, kvh, hd)
    q = rng.standard_normal((batch, rows, heads, hd)).astype(np.float32)
    pos = [0, 37, 5, 1][:batch]
    counts = [rows, rows - 3, 0, 200][:batch]
    _poison(pkg, backend, cache, [p + c for p, c in zip(pos, counts)])
    pick = {(b, t, h) for b in range(batch) for t in (0, 1, 31, 32, 130, rows - 4, rows - 1)
            for h in (0, heads - 1)}
    pick |= {(int(rng.integers(batch)), int(rng.integers(rows)), int(rng.integers(heads)))
             for _ in range(60)}
    at = tuple(np.array(sorted(pick)).T)
    behind = np.arange(rows) >= np.array(counts)[:, None]
    for pre, ph, ahead in ((None, None, 0), (prefix, pheld, 70)):
        got, lse = _attend(pkg, backend, q, cache, pos, counts, hd ** -0.5, pre, ahead)
        want, wl, tol, lt = attention(q, held, pos, counts, hd ** -0.5, ph, ahead, pick)
        _close(got[at], want[at], tol[at])
        _close(lse[at], wl[at], lt[at])
        assert (got[behind] == 0).all() and np.isfinite(got).all()


@gpu
@pytest.mark.parametrize("rows,batch,kvh,hd,most", [(1, 3, 2, 64, 2400), (6, 20, 3, 128, 1500),
                                                    (30, 2, 2, 64, 2400)])
def test_rows_that_are_not_there(backend, pkg, rows, batch, kvh, hd, most):
    # What q holds in rows behind counts reaches no other row: NaN, infinities
    # and large numbers there change no bit, with and without a prefix.
    rng = np.random.default_rng(rows)
    cache, _ = _filled(pkg, backend, rng, batch, most, kvh, hd)
    prefix, _ = _filled(pkg, backend, rng, 1, 500, kvh, hd)
    q = rng.standard_normal((batch, rows, kvh, hd)).astype(np.float32)
    counts = [(i * 7) % (rows + 1) for i in range(batch)]
    behind = np.arange(rows) >= np.array(counts)[:, None]
    pos = [most - rows - 31 * i for i in range(batch)]
    for pre, ahead in ((None, 0), (prefix, 500)):
        q[behind] = 0
        want = _attend(pkg, backend, q, cache, pos, counts, 0.125, pre, ahead)
        for fill in (np.nan, np.inf, -3e38, 1e4):
            q[behind] = fill
            got = _attend(pkg, backend, q, cache, pos, counts, 0.125, pre, ahead)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        assert (want[0][behind] == 0).all() and np.isneginf(want[1][behind]).all()


@gpu
@pytest.mark.parametrize("rows", [1, 4])
def test_attention_over_a_large_cache(backend, pkg, rows):
    # Codes of more than the caches hold, read past them (134 MB): every
    # sequence the same rows, so that one tells of all.
    rng = np.random.default_rng(rows)
    batch, kvh, hd, most = 64, 4, 128, 2048
    k, v = (_rows(rng, 1, most, kvh, hd, 1) for _ in range(2))
    held = Held(1, most, kvh, hd)
    held.write(k, v, [0], [most])
    cache = pkg.hip.Q8Cache(backend, batch, most, kvh, hd)
    for at in range(0, most, 256):
        part = [np.repeat(x[:, at:at + 256], batch, 0) for x in (k, v)]
        _write(pkg, backend, cache, *part, [at] * batch, None)
    q = np.repeat(rng.standard_normal((1, rows, 2 * kvh, hd)), batch, 0).astype(np.float32)
    got, lse = _attend(pkg, backend, q, cache, [most - rows] * batch, None, 0.1)
    want, wl, tol, lt = attention(q[:1], held, [most - rows], [rows], 0.1)
    _close(got[:1], want, tol)
    _close(lse[:1], wl, lt)
    assert (got == got[:1]).all() and (lse == lse[:1]).all()


@gpu
@pytest.mark.parametrize("rows", [1, 12])
def test_attention_and_nan(backend, pkg, rows):
    # A NaN row inside the attended ones and a NaN or infinite q make their
    # heads NaN and nothing else; no lse asked for.
    rng = np.random.default_rng(rows)
    batch, kvh, hd, n = 4, 2, 64, 70
    cache, held = _filled(pkg, backend, rng, batch, n, kvh, hd)
    bad = np.ones((batch, 1, kvh, hd), np.float32)
    bad[1, 0, 0, 3] = np.nan
    good = np.ones_like(bad)
    _write(pkg, backend, cache, bad, good, [40] * batch, None)
    held.write(bad, good, [40] * batch, [1] * batch)
    bad[1, 0, 0, 3] = 1
    bad[2, 0, 1, 5] = np.inf
    _write(pkg, backend, cache, good, bad, [41] * batch, None)
    held.write(good, bad, [41] * batch, [1] * batch)
    q = rng.standard_normal((batch, rows, 2 * kvh, hd)).astype(np.float32)
    q[0, 0, 1, 0] = np.nan
    q[3, 0, 2, 9] = np.inf
    pos = [n - rows] * batch
    got, _ = _attend(pkg, backend, q, cache, pos, None, 0.125, want_lse=False)
    want, _, tol, _ = attention(q, held, pos, [rows] * batch, 0.125)
    nan = np.zeros(q.shape[:3], bool)
    nan[1, :, :2] = nan[2, :, 2:] = True
    nan[0, 0, 1] = nan[3, 0, 2] = True
    assert np.isnan(got[nan]).all()
    _close(got[~nan], want[~nan], tol[~nan])


@gpu
def test_attention_past_32_bits(backend, pkg):
    # The last slot's V rows lie past 2^32 bytes of the buffer (4.9 GB).
    slots, most, kvh, hd = 6, 1 << 20, 6, 64
    cache = pkg.hip.Q8Cache(backend, slots, most, kvh, hd)
    rng = np.random.default_rng(8)
    n, at = 40, most - 50
    k, v = (_rows(rng, slots, n, kvh, hd, 2) for _ in range(2))
    _write(pkg, backend, cache, k, v, [at] * slots, None)
    gk, gv = _read(backend, cache, slots, n, [at] * slots, None)
    assert np.array_equal(gk, quantise(k)) and np.array_equal(gv, quantise(v))
    # Rows below `at` are zeros: each takes weight 1, relative to scores of
    # its own zero, as the formula says.
    q = rng.standard_normal((slots, 1, kvh, hd)).astype(np.float32)
    got, lse = _attend(pkg, backend, q, cache, [at + n - 1] * slots, None, 1.0)
    x = np.einsum("bhd,bnhd->bhn", q[:, 0].astype(np.float64), quantise(k))
    p = np.exp(x)
    want = np.einsum("bhn,bnhd->bhd", p, quantise(v)) / (p.sum(-1) + at)[..., None]
    # Of a million sums the kernel's own are at most a few thousand long.
    assert np.abs(lse[:, 0] - np.log(p.sum(-1) + at)).max() < 1e-3
    assert np.abs(got[:, 0] - want).max() < 1e-3 * np.abs(want).max()


@gpu
def test_step_in_a_graph_follows_its_live_lengths(pkg):
    # Write and attend captured once, replayed while pos and counts move, and
    # checked against the eager calls; two graphs share one workspace.
    h = pkg.hip
    be = h.Backend(0)
    try:
        rng = np.random.default_rng(3)
        batch, rows, heads, kvh, hd, most = 3, 4, 4, 2, 64, 3000
        held, pheld = Held(batch, most, kvh, hd), None
        cache = h.Q8Cache(be, batch, most, kvh, hd)
        prefix, pheld = _filled(pkg, be, rng, 1, 300, kvh, hd)
        first = [_rows(rng, batch, 2000, kvh, hd, 1) for _ in range(2)]
        _write(pkg, be, cache, *first, [0] * batch, None)
        held.write(*first, [0] * batch, [2000] * batch)
        n = batch * rows
        dk, dv, dq = be.zeros(n * kvh * hd), be.zeros(n * kvh * hd), be.zeros(n * heads * hd)
        out, out2 = be.zeros(n * heads * hd), be.zeros(n * heads * hd)
        dpos, dcnt, dlen = be.zeros(batch, np.uint32), be.zeros(batch, np.uint32), be.zeros(1, np.uint32)
        shape = h.AttnQ8(batch, rows, heads, heads * hd, heads * hd, 0.125, 0)
        size = max(h.attn_q8_workspace(shape, cache), h.attn_q8_workspace(shape, cache, prefix))
        ws = be.zeros(size // 4 + 1)
        graphs = []
        for _ in range(2):
            be.graph_begin()
            be.cache_write_q8(dk, dv, cache, batch, rows, kvh * hd, dpos, dcnt)
            be.attn_cached_q8(dq, cache, out, None, shape, dpos, dcnt, ws, size)
            be.attn_prefix_q8(dq, prefix, dlen, cache, out2, None, shape, dpos, dcnt, ws, size)
            graphs.append(be.graph_end())
        at = np.array([1990, 7, 500])
        for step in range(5):
            counts = np.array([[4, 2, 0], [1, 4, 3], [0, 0, 4], [4, 4, 4], [2, 1, 3]][step])
            k, v = (_rows(rng, batch, rows, kvh, hd, 1) for _ in range(2))
            q = rng.standard_normal((batch, rows, heads, hd)).astype(np.float32)
            ahead = [300, 0, 17, 200, 299][step]
            dk.upload(k), dv.upload(v), dq.upload(q)
            dpos.upload(at.astype(np.uint32)), dcnt.upload(counts.astype(np.uint32))
            dlen.upload(np.uint32([ahead]))
            graphs[step % 2].execute()
            held.write(k, v, at, counts)
            got = [o.download().reshape(q.shape) for o in (out, out2)]
            want, _, tol, _ = attention(q, held, at, counts, 0.125)
            _close(got[0], want, tol)
            want, _, tol, _ = attention(q, held, at, counts, 0.125, pheld, ahead)
            _close(got[1], want, tol)
            eager, _ = _attend(pkg, be, q, cache, at, counts, 0.125)
            assert np.array_equal(eager, got[0])
            be.synchronize()
            at = at + counts
        for g in graphs:
            g.close()
    finally:
        be.close()


@gpu
def test_same_call_twice_is_the_same(backend, pkg):
    rng = np.random.default_rng(11)
    cache, _ = _filled(pkg, backend, rng, 4, 2600, 2, 64)
    prefix, _ = _filled(pkg, backend, rng, 1, 900, 2, 64)
    q = rng.standard_normal((4, 5, 4, 64)).astype(np.float32)
    pos = [2500, 3, 1000, 40]
    for pre, ahead in ((None, 0), (prefix, 900)):
        a = _attend(pkg, backend, q, cache, pos, None, 0.125, pre, ahead)
        b = _attend(pkg, backend, q, cache, pos, None, 0.125, pre, ahead)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@gpu
@pytest.mark.parametrize("batch,rows,heads,kvh,hd,n", [(1, 1, 2, 2, 64, 50000), (2, 12, 2, 2, 64, 20000),
                                                      (1, 128, 16, 16, 128, 3000), (32, 64, 16, 16, 128, 500)])
def test_one_key_next_to_many(backend, pkg, batch, rows, heads, kvh, hd, n):
    # The first key weighs about as much as all others together, which weigh
    # the same: whatever a small weight loses is lost n times over.
    rng = np.random.default_rng(n)
    u = rng.standard_normal(hd).astype(np.float32)
    k = np.zeros((batch, n, kvh, hd), np.float32)
    v = np.ones_like(k)
    k[:, 0], v[:, 0] = u, 0
    q = np.broadcast_to(u / (u @ u), (batch, rows, heads, hd)).astype(np.float32)
    scale = float(np.float32(np.log(n) + 0.37))
    cache = pkg.hip.Q8Cache(backend, batch, n, kvh, hd)
    _write(pkg, backend, cache, k, v, [0] * batch, None)
    got, lse = _attend(pkg, backend, q, cache, [n - rows] * batch, None, scale)
    x0 = scale * (quantise(u[None])[0] @ q[0, 0, 0].astype(np.float64))
    others = n - rows + np.arange(rows)
    want = others / (others + np.exp(x0))
    # The score is off by (hd + 8) 2^-23 of its products' magnitudes (their sum is near x0 < 12)
    # and as an exponent of 2 by 2^-22; a weight by 2^-22; a wave adds n / 32 /
    # 4 tiles in f32.
    tol = 12 * (hd + 8) * 2.0 ** -23 + 12 * 2.0 ** -22 + 2.0 ** -21 + n / 128 * 2.0 ** -24
    assert np.abs(got / want[:, None, None] - 1).max() <= tol
    assert np.abs(lse - np.log(others + np.exp(x0))[:, None]).max() <= tol + 2.0 ** -20


@gpu
def test_backends_side_by_side(pkg):
    # Two backends' calls (streams and workspaces of their own) under way at
    # once over one cache's rows give what each gives alone.
    h = pkg.hip
    a, b = h.Backend(0), h.Backend(0)
    try:
        rng = np.random.default_rng(21)
        batch, heads, kvh, hd, most = 8, 8, 4, 128, 3000
        cache, _ = _filled(pkg, a, rng, batch, most, kvh, hd)
        a.synchronize()
        seen = h.Q8Cache(b, batch, most, kvh, hd, data=cache.data)
        q = [rng.standard_normal((batch, rows, heads, hd)).astype(np.float32) for rows in (1, 6)]
        alone = [_attend(pkg, a, x, cache, [most - 6] * batch, None, 0.1)[0] for x in q]
        calls = []
        for be, c, x in ((a, cache, q[0]), (b, seen, q[1])):
            rows = x.shape[1]
            shape = h.AttnQ8(batch, rows, heads, heads * hd, heads * hd, 0.1, 0)
            size = h.attn_q8_workspace(shape, c)
            calls.append((be, be.tensor(x), c, be.zeros(x.size), shape, _u32(be, [most - 6] * batch),
                          be.zeros(size // 4 + 1), size))
        a.synchronize(), b.synchronize()
        for _ in range(20):
            for be, dq, c, out, shape, pos, ws, size in calls:
                be.attn_cached_q8(dq, c, out, None, shape, pos, None, ws, size)
        for (be, _, _, out, *_), x, want in zip(calls, q, alone):
            assert np.array_equal(out.download().reshape(x.shape), want)
    finally:
        b.close()
        a.close()


# ---- refusals ----------------------------------------------------------------


def _stand_in(pkg):
    """A handle to zeroed memory in a backend's place: the checks run before
    anything of the backend is used, and without a device."""
    pkg.hip.load()
    mem = (C.c_char * 8192)()
    return mem, C.cast(mem, C.c_void_p)


def _cache_c(h, data=1 << 20, slots=4, max_rows=64, kv_heads=2, head_dim=64):
    return h.Q8CacheC(data, slots, max_rows, kv_heads, head_dim)


def test_rows_refusals(pkg):
    h = pkg.hip
    lib, (mem, be) = h.load(), _stand_in(pkg)
    x, bad = C.c_void_p(1 << 21), h.InvalidArgument.code

    def write(cache, batch=4, rows=2, stride=128, pos=x, k=x, v=x, backend=be):
        return lib.akh_cache_write_q8(backend, k, v, cache, batch, rows, stride, pos, None)

    def read(cache, batch=4, rows=2, stride=128, pos=x):
        return lib.akh_cache_read_q8(be, cache, x, x, batch, rows, stride, pos, None)

    good = _cache_c(h)
    for call in (write, read):
        assert call(_cache_c(h, data=None)) == bad
        assert call(_cache_c(h, data=(1 << 20) + 8)) == bad
        assert call(_cache_c(h, head_dim=129)) == bad
        assert call(_cache_c(h, head_dim=0)) == bad
        assert call(_cache_c(h, max_rows=(1 << 30) + 1)) == bad
        assert call(good, batch=5) == bad
        assert call(good, stride=127) == bad
        assert call(good, pos=None) == bad
        assert call(_cache_c(h, slots=1 << 20), batch=1 << 20, rows=1 << 20) == bad
        # A grid of 2^24 blocks or more.
        assert call(_cache_c(h, slots=1 << 24), batch=1 << 24, rows=1) == bad
        assert call(_cache_c(h, slots=1 << 24), batch=1 << 24, rows=4) == bad
        assert call(good, batch=0) == 0 and call(good, rows=0) == 0
    assert write(good, k=None) == bad and write(good, v=None) == bad
    assert write(good, backend=None) == bad
    assert lib.akh_cache_read_q8(be, good, None, None, 4, 2, 128, x, None) == 0


def test_attention_refusals(pkg):
    h = pkg.hip
    lib, (mem, be) = h.load(), _stand_in(pkg)
    x, bad = C.c_void_p(1 << 21), h.InvalidArgument.code

    def call(cache=None, prefix=None, batch=4, rows=2, heads=4, q_stride=256, out_stride=256,
             scale=0.125, q=x, out=x, pos=x, plen=x, ws=C.c_void_p(1 << 22), size=1 << 40):
        s = h.AttnQ8(batch, rows, heads, q_stride, out_stride, scale, 0)
        cache = cache or _cache_c(h)
        if prefix is None:
            return lib.akh_attn_cached_q8(be, q, cache, out, None, s, pos, None, ws, size)
        return lib.akh_attn_prefix_q8(be, q, prefix, plen, cache, out, None, s, pos, None, ws, size)

    for prefix in (None, _cache_c(h, slots=1, max_rows=1000)):
        for kw in ({"batch": 5}, {"heads": 3}, {"heads": 0}, {"q_stride": 255},
                   {"out_stride": 255}, {"scale": float("nan")}, {"scale": float("inf")},
                   {"q": None}, {"out": None}, {"pos": None}, {"rows": 1 << 22}, {"rows": 1 << 20},
                   {"cache": _cache_c(h, data=None)}, {"cache": _cache_c(h, data=24)},
                   {"cache": _cache_c(h, kv_heads=3)}, {"cache": _cache_c(h, head_dim=200)}):
            assert call(prefix=prefix, **kw) == bad, kw
        assert call(prefix=prefix, batch=0) == 0 and call(prefix=prefix, rows=0) == 0
    good = _cache_c(h, slots=1)
    assert call(prefix=_cache_c(h, data=None)) == bad
    assert call(prefix=_cache_c(h, head_dim=128)) == bad
    assert call(prefix=_cache_c(h, kv_heads=1)) == bad
    assert call(prefix=good, plen=None) == bad
    # A workspace that is missing, short or unaligned, where one is needed.
    s, n = h.AttnQ8(1, 1, 4, 512, 512, 0.1, 0), C.c_size_t()
    long = _cache_c(h, slots=1, max_rows=1 << 20, head_dim=128)
    assert lib.akh_attn_q8_workspace(C.byref(s), C.byref(long), None, C.byref(n)) == 0
    if n.value:
        kw = dict(cache=long, batch=1, rows=1, q_stride=512, out_stride=512)
        assert call(ws=None, **kw) == bad
        assert call(size=n.value - 1, **kw) == bad
        assert call(ws=C.c_void_p((1 << 22) + 4), **kw) == bad
    assert lib.akh_attn_q8_workspace(None, C.byref(long), None, C.byref(n)) == bad
