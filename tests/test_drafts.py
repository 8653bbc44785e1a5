"""Drafted tokens served from an 8-bit cache: the calls of a step together
(akh_cache_write_q8, akh_attn_prefix_q8 or akh_attn_cached_q8, akh_matmul,
akh_verify_drafts), captured in one graph, step after step, with a cache that
is cut back to the tokens that were kept.

The model is one attention layer over made-up tables: token x at place p has
q, k and v rows ``table[x] + place[p]``, and logits out @ W.  Every step is
checked against the definitions in 64 bits, which follow the device's tokens.
"""

import numpy as np
import pytest

from test_q8 import Held, _bounds, _close, attention, quantise  # noqa: F401
from test_verify import END, verify

gpu = pytest.mark.gpu

HEADS, KVH, HD, VOCAB, BATCH, DRAFTS = 4, 2, 64, 301, 3, 3
PLACES = 400


class Model:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.tables = {}
        for name, heads in (("q", HEADS), ("k", KVH), ("v", KVH)):
            self.tables[name] = (rng.standard_normal((VOCAB, heads, HD)).astype(np.float32),
                                 rng.standard_normal((PLACES, heads, HD)).astype(np.float32))
        self.w = (rng.standard_normal((HEADS * HD, VOCAB)) * 0.6).astype(np.float32)

    def rows(self, name, tokens, places):
        token, place = self.tables[name]
        return token[tokens] + place[places]


class Serving:
    """A batch of sequences behind a shared prefix (or none), on the device."""

    def __init__(self, pkg, be, model, prompt, tails, temperature, drawn):
        h = pkg.hip
        self.be, self.model, self.temperature = be, model, temperature
        self.ahead = len(prompt)
        self.rows = rows = DRAFTS + 1
        n = BATCH * rows
        self.cache = h.Q8Cache(be, BATCH, 200, KVH, HD)
        self.held = Held(BATCH, 200, KVH, HD)
        self.prefix = self.pheld = None
        up = lambda x: be.tensor(np.ascontiguousarray(x))  # noqa: E731
        if self.ahead:
            self.prefix, self.pheld = h.Q8Cache(be, 1, self.ahead, KVH, HD), Held(1, self.ahead, KVH, HD)
            kv = [model.rows(x, prompt, np.arange(self.ahead))[None] for x in "kv"]
            be.cache_write_q8(up(kv[0]), up(kv[1]), self.prefix, 1, self.ahead, KVH * HD,
                              be.zeros(1, np.uint32))
            self.pheld.write(*kv, [0], [self.ahead])
        # The sequences' own prompts but for their last tokens, padded to the longest.
        self.pos = np.array([len(t) - 1 for t in tails])
        padded = np.zeros((BATCH, self.pos.max()), int)
        for b, t in enumerate(tails):
            padded[b, :len(t) - 1] = t[:-1]
        kv = [model.rows(x, padded, self.ahead + np.arange(padded.shape[1])) for x in "kv"]
        be.cache_write_q8(up(kv[0]), up(kv[1]), self.cache, BATCH, padded.shape[1], KVH * HD,
                          be.zeros(BATCH, np.uint32), up(self.pos.astype(np.uint32)))
        self.held.write(*kv, [0] * BATCH, self.pos)
        self.last = np.array([t[-1] for t in tails])

        self.q, self.k, self.v = be.zeros(n * HEADS * HD), be.zeros(n * KVH * HD), be.zeros(n * KVH * HD)
        self.dpos, self.counts, self.drafts = (be.zeros(BATCH, np.uint32) for _ in range(3))
        self.plen = up(np.uint32([self.ahead]))
        self.out, self.logits = be.zeros(n * HEADS * HD), be.zeros(n * VOCAB)
        self.lse = be.zeros(n * HEADS)
        self.w = up(model.w)
        self.tokens = be.zeros(BATCH * DRAFTS, np.uint32)
        self.draft = be.zeros(BATCH * DRAFTS * VOCAB) if drawn else None
        self.uniforms = be.zeros(BATCH * rows * 2)  # of 64 bits
        self.out_tokens, self.kept = be.zeros(n, np.uint32), be.zeros(BATCH, np.uint32)
        shape = h.AttnQ8(BATCH, rows, HEADS, HEADS * HD, HEADS * HD, HD ** -0.5, 0)
        size = h.attn_q8_workspace(shape, self.cache, self.prefix)
        vsize = h.verify_drafts_workspace(BATCH, DRAFTS, VOCAB)
        ws = self.ws = be.tensor(np.full(max(size, vsize), 0xFF, np.uint8))  # both calls' in turn
        mm = h.MatMulMeta(n, VOCAB, HEADS * HD)
        meta = be.meta(mm)
        self.meta = meta

        def step():
            be.cache_write_q8(self.k, self.v, self.cache, BATCH, rows, KVH * HD, self.dpos, self.counts)
            if self.prefix is None:
                be.attn_cached_q8(self.q, self.cache, self.out, self.lse, shape, self.dpos,
                                  self.counts, ws, size)
            else:
                be.attn_prefix_q8(self.q, self.prefix, self.plen, self.cache, self.out, self.lse,
                                  shape, self.dpos, self.counts, ws, size)
            be.matmul(self.out, self.w, self.logits, mm, meta)
            be.verify_drafts(self.logits, self.draft, self.tokens, BATCH, DRAFTS, VOCAB,
                             self.out_tokens, self.kept, None, temperature, self.drafts,
                             self.uniforms, ws, vsize)

        be.graph_begin()
        step()
        self.graph = be.graph_end()
        self.eager = step

    def step(self, proposed, drafted, draft_logits, uniforms, eager):
        """One step over proposed [BATCH, DRAFTS] of which the first drafted[b]
        are drafts; returns the kept tokens of each sequence."""
        be, rows = self.be, self.rows
        tokens = np.concatenate([self.last[:, None], proposed], 1)
        places = self.ahead + self.pos[:, None] + np.arange(rows)
        q, k, v = (self.model.rows(x, tokens, places) for x in "qkv")
        for d, x in ((self.q, q), (self.k, k), (self.v, v)):
            d.upload(x)
        self.dpos.upload(self.pos.astype(np.uint32))
        self.counts.upload((drafted + 1).astype(np.uint32))
        self.drafts.upload(drafted.astype(np.uint32))
        self.tokens.upload(proposed.astype(np.uint32))
        if self.draft is not None:
            self.draft.upload(draft_logits)
        self.uniforms.upload(uniforms)
        self.eager() if eager else self.graph.execute()

        self.held.write(k, v, self.pos, drafted + 1)
        out, lse, tol, ltol = attention(q, self.held, self.pos, drafted + 1, HD ** -0.5, self.pheld,
                                        self.ahead)
        got = self.out.download().reshape(out.shape)
        _close(got, out, tol)
        _close(self.lse.download().reshape(lse.shape), lse, ltol)
        # The choice is the rule's on the logits the device has.
        logits = self.logits.download().reshape(BATCH, rows, VOCAB)
        want = verify(logits, draft_logits if self.draft is not None else None,
                      proposed.astype(np.uint32), self.temperature, uniforms, drafted)
        kept = self.kept.download(np.uint32, BATCH)
        chosen = self.out_tokens.download(np.uint32, BATCH * rows).reshape(BATCH, rows)
        assert np.array_equal(kept, want[1]) and np.array_equal(chosen, want[0])
        assert (chosen[np.arange(rows) >= kept[:, None]] == END).all()
        # Refused drafts' rows stay behind pos and are written over by the next step.
        self.pos = self.pos + kept
        self.last = chosen[np.arange(BATCH), kept - 1].astype(int)
        return [chosen[b, :kept[b]].tolist() for b in range(BATCH)]


def prompts(rng, ahead):
    return (rng.integers(0, VOCAB, ahead),
            [rng.integers(0, VOCAB, n) for n in (1, 40, 17)])


def one_by_one(model, prompt, tails, steps):
    """Tokens that greedy decoding without drafts gives, in 64 bits, and the
    least distance of a largest logit from the next."""
    told, margin = [], np.inf
    for tail in tails:
        line, new = list(prompt) + list(tail), []
        for _ in range(steps):
            k, v = (quantise(model.rows(x, np.array(line), np.arange(len(line)))) for x in "kv")
            q = model.rows("q", line[-1], len(line) - 1).astype(np.float64)
            out = np.zeros((HEADS, HD))
            for h in range(HEADS):
                x = k[:, h * KVH // HEADS] @ q[h] * HD ** -0.5
                p = np.exp(x - x.max())
                out[h] = p @ v[:, h * KVH // HEADS] / p.sum()
            logits = out.reshape(-1) @ model.w.astype(np.float64)
            top = np.sort(logits)[-2:]
            margin = min(margin, top[1] - top[0])
            new.append(int(logits.argmax()))
            line.append(new[-1])
        told.append(new)
    return told, margin


@gpu
@pytest.mark.parametrize("ahead", [0, 1, 77])
def test_greedy_drafts_change_no_token(pkg, ahead):
    # Whatever is proposed, the tokens are those of decoding one by one.
    rng = np.random.default_rng(ahead)
    model = Model(7)
    prompt, tails = prompts(rng, ahead)
    steps = 24
    told, margin = one_by_one(model, prompt, tails, steps + DRAFTS + 1)
    # Scores of 64 roundings of both signs are some 8 * 2^-24 * 20 = 1e-5 off, out's
    # elements with them, logits (256 of those times 0.6) 1e-4: far from the
    # closest two here.
    assert margin > 1e-2
    be = pkg.hip.Backend(0)
    try:
        s = Serving(pkg, be, model, prompt, tails, 0.0, False)
        said = [[] for _ in range(BATCH)]
        i = 0
        while min(map(len, said)) < steps:
            drafted = np.array([(i + b) % (DRAFTS + 1) for b in range(BATCH)])
            ahead_of = np.array([(told[b] + [0] * 99)[len(said[b]):len(said[b]) + DRAFTS]
                                 for b in range(BATCH)])
            wrong = rng.random((BATCH, DRAFTS)) < 0.3
            proposed = np.where(wrong, rng.integers(0, VOCAB, wrong.shape), ahead_of)
            for b, new in enumerate(s.step(proposed, drafted, None, np.zeros((BATCH, s.rows)),
                                           eager=i % 5 == 3)):
                said[b] += new
            i += 1
        for b in range(BATCH):
            n = min(len(said[b]), len(told[b]))
            assert said[b][:n] == told[b][:n]
        # Rows of tokens that were kept are in the cache, and only those count.
        rows = [model.rows(x, np.array(list(tails[1]) + said[1])[:s.pos[1]],
                           ahead + np.arange(s.pos[1])) for x in "kv"]
        k, v = (be.zeros(int(s.pos[1]) * KVH * HD) for _ in range(2))
        first = be.zeros(BATCH, np.uint32)
        wide = [be.zeros(BATCH * int(s.pos[1]) * KVH * HD) for _ in range(2)]
        be.cache_read_q8(s.cache, *wide, BATCH, int(s.pos[1]), KVH * HD, first)
        for x, w in zip(rows, wide):
            got = w.download().reshape(BATCH, -1, KVH, HD)[1]
            assert np.array_equal(got, quantise(x))
        s.graph.close()
    finally:
        be.close()


@gpu
@pytest.mark.parametrize("ahead", [0, 130])
@pytest.mark.parametrize("drawn", [False, True])
def test_sampled_drafts(pkg, ahead, drawn):
    rng = np.random.default_rng(ahead + drawn)
    model = Model(9)
    be = pkg.hip.Backend(0)
    try:
        s = Serving(pkg, be, model, *prompts(rng, ahead), 0.9, drawn)
        kept = 0
        for i in range(20):
            logits = (rng.standard_normal((BATCH, DRAFTS, VOCAB)) * 1.5).astype(np.float32)
            noise = -np.log(-np.log(rng.random(logits.shape)))
            proposed = (logits / 0.9 + noise).argmax(-1)
            drafted = rng.integers(0, DRAFTS + 1, BATCH)
            new = s.step(proposed, drafted, logits, rng.random((BATCH, s.rows)), eager=i % 4 == 1)
            kept += sum(map(len, new))
        assert kept >= 20 * BATCH
        s.graph.close()
    finally:
        be.close()
