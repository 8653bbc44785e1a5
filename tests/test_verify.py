"""Verification of drafted tokens (akh_verify_drafts) against its rule in 64
bits.  Tokens are whole numbers and have to be equal: both sides compute
probabilities in 64 bits, so a draw would have to fall within about 1e-12 of
a border of the cumulative weights (50257 of them at most) to be resolved
differently."""

import ctypes as C

import numpy as np
import pytest

gpu = pytest.mark.gpu
END = 0xFFFFFFFF


# ---- the rule in 64 bits ---------------------------------------------------


def softmax(l, temperature):
    """Probabilities of logits; NaN has none, all zero where no weight is left."""
    l = l.astype(np.float64)
    with np.errstate(all="ignore"):
        top = np.nanmax(l) if not np.isnan(l).all() else -np.inf
        w = np.exp((l - top) / float(np.float32(temperature)))
        w = np.where(w > 0, w, 0.0)
        return w / w.sum() if w.sum() > 0 else np.zeros_like(w)


def first_max(l):
    ok = ~np.isnan(l)
    return int(np.argmax(np.where(ok, l, -np.inf) == l[ok].max())) if ok.any() else 0


def draw(weights, u):
    """The lowest id whose cumulative weight exceeds u times the total."""
    cum = np.cumsum(weights)
    hit = np.nonzero((cum > u * cum[-1]) & (weights > 0))[0]
    return int(hit[0]) if hit.size else int(np.nonzero(weights > 0)[0][-1])


def verify(target, draft, tokens, temperature, uniforms, counts):
    """(tokens [batch, rows + 1], counts, chance) of speculative sampling."""
    batch, rows = tokens.shape
    n = target.shape[-1]
    out = np.full((batch, rows + 1), END, np.uint32)
    kept, chance = np.zeros(batch, np.uint32), np.zeros((batch, rows))
    for b in range(batch):
        c = min(int(counts[b]), rows)
        refused = c
        for t in range(c):
            x = int(tokens[b, t])
            if temperature <= 0:
                ok = x == first_max(target[b, t])
                chance[b, t] = ok
            else:
                p = softmax(target[b, t], temperature)
                px = p[x] if x < n else 0.0
                qx = 1.0 if draft is None or x >= n else softmax(draft[b, t], temperature)[x]
                ok = uniforms[b, t] * qx < px
                chance[b, t] = 0.0 if px == 0 else 1.0 if qx == 0 else min(1.0, px / qx)
            if not ok:
                refused = min(refused, t)
        row = target[b, refused]
        last = first_max(row)
        if temperature > 0:
            p = softmax(row, temperature)
            q = np.zeros(n)
            if refused < c:
                if draft is not None:
                    q = softmax(draft[b, refused], temperature)
                elif tokens[b, refused] < n:
                    q[tokens[b, refused]] = 1.0
            w = np.maximum(p - q, 0.0)
            w = w if w.sum() > 0 else p
            if w.sum() > 0:
                last = draw(w, uniforms[b, rows])
        out[b, :refused] = tokens[b, :refused]
        out[b, refused] = last
        kept[b] = refused + 1
    return out, kept, chance


def test_rule_draws_from_the_target():
    # Whatever the drafts' distribution, the first token is the target's draw.
    rng = np.random.default_rng(0)
    n, trials = 5, 20000
    target, draft = rng.standard_normal((1, 2, n)) * 1.5, rng.standard_normal((1, 1, n)) * 1.5
    for d, temperature in ((draft, 0.7), (None, 1.3)):
        q = softmax(draft[0, 0], temperature)
        tokens = rng.choice(n, size=(trials, 1), p=q) if d is not None else np.full((trials, 1), 2)
        u = rng.random((trials, 2))
        out, kept, chance = verify(np.repeat(target, trials, 0),
                                   None if d is None else np.repeat(d, trials, 0), tokens,
                                   temperature, u, np.ones(trials))
        p = softmax(target[0, 0], temperature)
        seen = np.bincount(out[:, 0], minlength=n) / trials
        # Five standard deviations of a frequency.
        assert (np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / trials)).all()
        rate = np.minimum(p, q).sum() if d is not None else p[2]
        assert abs((kept == 2).mean() - rate) <= 5 * np.sqrt(rate * (1 - rate) / trials) + 1e-12


# ---- the device ------------------------------------------------------------


def run(pkg, be, target, draft, tokens, temperature, uniforms, counts, want_chance=True):
    h = pkg.hip
    batch, rows = tokens.shape
    n = target.shape[-1]
    up = lambda a, t: be.tensor(np.ascontiguousarray(a, t))  # noqa: E731
    size = h.verify_drafts_workspace(batch, rows, n)
    ws = be.tensor(np.full(size, 0xFF, np.uint8))
    out, kept = be.zeros(batch * (rows + 1), np.uint32), be.zeros(batch, np.uint32)
    chance = be.tensor(np.full(max(1, batch * rows), 9.0, np.float32)) if want_chance else None
    be.verify_drafts(up(target, np.float32), None if draft is None else up(draft, np.float32),
                     up(tokens, np.uint32), batch, rows, n, out, kept, chance,
                     temperature=temperature, counts=None if counts is None else up(counts, np.uint32),
                     uniforms=None if uniforms is None else up(uniforms, np.float64),
                     workspace=ws, workspace_bytes=size)
    return (out.download(np.uint32, batch * (rows + 1)).reshape(batch, rows + 1),
            kept.download(np.uint32, batch),
            chance.download(np.float32, batch * rows).reshape(batch, rows) if want_chance else None)


def check(pkg, be, target, draft, tokens, temperature, uniforms, counts):
    got = run(pkg, be, target, draft, tokens, temperature, uniforms, counts)
    want = verify(target, draft, tokens, temperature, uniforms,
                  np.full(len(tokens), END) if counts is None else counts)
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])
    # One rounding to 32 bits of a quotient exact to about 1e-12.
    assert (np.abs(got[2] - want[2]) <= 2.0 ** -24 * want[2] + 1e-12).all()
    return want


def make(rng, batch, rows, n, one_hot=False, near=0.7, spread=2.5):
    target = (rng.standard_normal((batch, rows + 1, n)) * spread).astype(np.float32)
    draft = (target[:, :rows] + rng.standard_normal((batch, rows, n)) * near).astype(np.float32)
    noise = -np.log(-np.log(rng.random((batch, rows, n))))
    tokens = (draft + noise).argmax(-1).astype(np.uint32)
    return target, None if one_hot else draft, tokens, rng.random((batch, rows + 1))


@gpu
@pytest.mark.parametrize("batch,rows,n", [(1, 1, 1), (3, 1, 2), (5, 4, 97), (2, 7, 4095), (4, 3, 4096),
                                          (3, 2, 4097), (2, 5, 50257), (9, 8, 12289), (1, 300, 50)])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0, 3.0])
@pytest.mark.parametrize("one_hot", [False, True])
def test_matches_the_rule(backend, pkg, batch, rows, n, temperature, one_hot):
    rng = np.random.default_rng(batch * 1000 + n + one_hot)
    target, draft, tokens, u = make(rng, batch, rows, n, one_hot)
    counts = np.array([(i * 3) % (rows + 2) for i in range(batch)])
    check(pkg, backend, target, draft, tokens, temperature, u, counts)
    check(pkg, backend, target, draft, tokens, temperature, u, None)


@gpu
@pytest.mark.parametrize("batch,rows,n,temperature", [(2, 1, 1 << 20, 1.0), (1, 2, (1 << 20) - 1, 0.6),
                                                      (3, 1, 65537, 1.0), (2, 1, 1 << 20, 0.0),
                                                      (1, 1024, 33, 1.0), (300, 2, 70, 1.0)])
def test_largest_sizes(backend, pkg, batch, rows, n, temperature):
    rng = np.random.default_rng(n + batch)
    target, draft, tokens, u = make(rng, batch, rows, n, near=0.3)
    check(pkg, backend, target, draft, tokens, temperature, u, None)
    # Draws near the end of the walk, and drafts that are all refused.
    u[:, rows] = 1 - 2.0 ** -20
    tokens[:] = (target[:, :rows].argmin(-1)).astype(np.uint32)
    check(pkg, backend, target, draft, tokens, temperature, u, None)
    check(pkg, backend, target, None, tokens, temperature, u, None)


@gpu
def test_accepts_all_and_none(backend, pkg):
    rng = np.random.default_rng(2)
    target, draft, tokens, u = make(rng, 6, 4, 3000, near=0.0)  # p == q: all accepted
    want = check(pkg, backend, target, draft, tokens, 1.0, u, None)
    assert (want[1] == 5).all()
    # The draft is sure of what the target excludes: none accepted.
    target[:, 0, :10] = -np.inf
    draft[:, 0] = -np.inf
    draft[:, 0, 3] = 1.0
    tokens[:, 0] = 3
    want = check(pkg, backend, target, draft, tokens, 1.0, u, None)
    assert (want[1] == 1).all() and (want[0][:, 0] >= 10).all()
    # Draws at both ends of [0, 1).
    for end in (0.0, np.nextafter(1.0, 0.0)):
        u[:] = end
        check(pkg, backend, target, draft, tokens, 1.0, u, None)


@gpu
def test_ties_go_to_the_lowest_id(backend, pkg):
    target = np.zeros((2, 3, 9000), np.float32)
    target[0, :, [4000, 4097, 8999]] = 2.0
    tokens = np.array([[4000, 4097], [0, 1]], np.uint32)
    want = check(pkg, backend, target, None, tokens, 0.0, np.zeros((2, 3)), None)
    assert list(want[0][0]) == [4000, 4000, END] and list(want[0][1]) == [0, 0, END]
    check(pkg, backend, target, None, tokens, 1.0, np.full((2, 3), 0.25), None)


@gpu
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_rows_of_nan_and_infinities(backend, pkg, temperature):
    rng = np.random.default_rng(4)
    target, draft, tokens, u = make(rng, 9, 2, 5000)
    nan, inf = np.nan, np.inf
    target[0, 0, ::3] = nan          # some
    target[1, 0] = nan               # all
    target[2, 0] = -inf              # nothing possible
    target[3, 0, [17, 4500]] = inf   # an infinite maximum
    target[4, 0, 7:] = -inf          # a few possible
    draft[5, 0] = nan                # a draft without a distribution
    draft[6, 0, 1::2] = -inf
    tokens[7, 0] = 5000              # no such id
    tokens[8, 0] = END
    check(pkg, backend, target, draft, tokens, temperature, u, None)
    check(pkg, backend, target, None, tokens, temperature, u, None)


@gpu
@pytest.mark.parametrize("temperature", [np.inf, 3e38, 1e-38, 1e-45])
def test_temperatures_at_the_ends(backend, pkg, temperature):
    # Hot: all numbers above -infinity alike; cold: the maxima alone.
    rng = np.random.default_rng(12)
    target, draft, tokens, u = make(rng, 6, 3, 5000)
    target[:3, :, 1::2] = -np.inf
    draft[3:, :, ::3] = np.nan
    target[:, :, [7, 4999]] = target.max()
    check(pkg, backend, target, draft, tokens, temperature, u, None)
    check(pkg, backend, target, None, tokens, temperature, u, None)


@gpu
def test_without_drafts_it_samples(backend, pkg, ora):
    # rows = 0 (or counts 0) draws from the row itself, as the sampler's
    # temperature does, though not in the sampler's order of ids.
    rng = np.random.default_rng(6)
    target, draft, tokens, u = make(rng, 5, 0, 700)
    got = run(pkg, backend, target, None, tokens, 0.9, u, None)
    want = verify(target, None, tokens, 0.9, u, np.zeros(5))
    assert np.array_equal(got[0], want[0]) and (got[1] == 1).all()
    # Greedy agrees with akh_argmax_rows.
    got = run(pkg, backend, target, None, tokens, 0.0, None, None, want_chance=False)
    out = backend.zeros(5, np.uint32)
    backend.argmax_rows(backend.tensor(target), 5, 700, out)
    assert np.array_equal(got[0][:, 0], out.download(np.uint32, 5))


@gpu
def test_in_a_graph(pkg):
    h = pkg.hip
    be = h.Backend(0)
    try:
        rng = np.random.default_rng(7)
        batch, rows, n = 4, 3, 20000
        target, draft, tokens, u = make(rng, batch, rows, n)
        bufs = [be.tensor(x) for x in (target, draft, tokens, u)]
        counts = be.zeros(batch, np.uint32)
        out, kept = be.zeros(batch * (rows + 1), np.uint32), be.zeros(batch, np.uint32)
        size = h.verify_drafts_workspace(batch, rows, n)
        ws = be.zeros(size // 4 + 1)
        be.graph_begin()
        be.verify_drafts(*bufs[:3], batch, rows, n, out, kept, temperature=0.9, counts=counts,
                         uniforms=bufs[3], workspace=ws, workspace_bytes=size)
        g = be.graph_end()
        for step in range(4):
            target, draft, tokens, u = make(rng, batch, rows, n)
            for d, x in zip(bufs, (target, draft, tokens, u)):
                d.upload(x)
            c = rng.integers(0, rows + 1, batch).astype(np.uint32)
            counts.upload(c)
            g.execute()
            want = verify(target, draft, tokens, 0.9, u, c)
            assert np.array_equal(out.download(np.uint32, batch * (rows + 1)).reshape(batch, -1), want[0])
            assert np.array_equal(kept.download(np.uint32, batch), want[1])
            again = run(pkg, be, target, draft, tokens, 0.9, u, c)
            assert np.array_equal(again[0], want[0])
            be.synchronize()
        g.close()
    finally:
        be.close()


def test_refusals(pkg):
    h = pkg.hip
    lib = h.load()
    mem = (C.c_char * 8192)()  # zeroed memory in a backend's place: checks run first
    be, x, bad = C.cast(mem, C.c_void_p), C.c_void_p(1 << 21), h.InvalidArgument.code

    def call(target=x, draft=x, tokens=x, batch=2, rows=3, n=100, temperature=1.0, uniforms=x,
             out=x, kept=x, ws=x, size=1 << 40, backend=be):
        return lib.akh_verify_drafts(backend, target, draft, tokens, batch, rows, n, temperature,
                                     None, uniforms, out, kept, None, ws, size)

    need = h.verify_drafts_workspace(2, 3, 100)
    for kw in ({"backend": None}, {"target": None}, {"tokens": None}, {"n": 0},
               {"n": (1 << 20) + 1}, {"rows": 1025}, {"batch": (1 << 20) + 1},
               {"temperature": float("nan")}, {"uniforms": None}, {"out": None}, {"kept": None},
               {"ws": None}, {"ws": C.c_void_p((1 << 21) + 8)}, {"size": need - 1},
               {"batch": 1 << 20, "rows": 1024, "n": 1 << 20},
               {"batch": 1 << 13, "rows": 1024, "n": 100}):
        assert call(**kw) == bad, kw
    assert call(batch=0) == 0
    with pytest.raises(h.InvalidArgument):
        h.verify_drafts_workspace(1, 1, 0)


def test_no_sequences_need_no_workspace(pkg):
    h = pkg.hip
    mem = (C.c_char * 8192)()  # zeroed memory in a backend's place: nothing of it is used
    be, x = C.cast(mem, C.c_void_p), C.c_void_p(1 << 21)
    assert h.verify_drafts_workspace(0, 3, 100) == 0
    for temperature in (0.0, 1.0):
        assert h.load().akh_verify_drafts(be, x, x, x, 0, 3, 100, temperature, None, x, x, x, None,
                                          None, 0) == 0
