"""Operator cases: serving drafted tokens from an 8-bit KV cache.

A case names one operator and its sizes:

* ``cache``: K and V rows, taken out of a fused QKV projection's output, are
  quantised into an 8-bit cache and read back as the values they then hold;
* ``read``: a stretch of a filled 8-bit cache is read back (cache hand-over);
* ``attn``: each sequence's newest rows attend to its own 8-bit cache;
* ``prefix``: the same, with a prefix that all sequences share before their
  own rows;
* ``verify``: drafted tokens against the target's logits from given uniforms.

An 8-bit cache is one buffer: K codes, V codes ([slots][kv_heads][cap][row])
and their exponents ([slots][kv_heads][cap], int8 as well), where ``row`` is
64 bytes for heads of up to 64 and 128 beyond, ``cap`` the rows rounded up to
32, and a value is code * 2^exponent.

With ``own`` false the operators are computed in their plain form from the
same buffers; with ``own`` true by the library's kernels, queued on the
backend's stream, which neither waits for torch's nor is waited for by it: a
state's first pass waits for the device, so that its inputs are there and
nothing of torch's still uses the memory of its outputs; whoever reads a
pass's outputs by torch, or drops a state, synchronises the device before.
"""

import ctypes
import importlib

import numpy as np
import torch

own = False

_backend = None


def listed():
    return [
        # A decode step's rows of a serving batch: one row per sequence.
        {"name": "step_rows", "kind": "cache", "batch": 32, "rows": 1, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "max_rows": 512, "ragged": False},
        # Prompts of uneven lengths going into the cache after their prefill.
        {"name": "prompt_rows", "kind": "cache", "batch": 8, "rows": 2040, "heads": 16,
         "kv_heads": 16, "head_dim": 128, "max_rows": 2048, "ragged": True},
        # A cache handed over to an fp32 consumer.
        {"name": "hand_over", "kind": "read", "batch": 8, "rows": 449, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "max_rows": 512, "ragged": True},
        # One user's chat: latency alone counts.
        {"name": "chat", "kind": "attn", "batch": 1, "rows": 1, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "length": 301, "ragged": False, "drafts": False},
        # A full serving batch near the end of a 512-token context, with
        # sequences of every length.
        {"name": "batch", "kind": "attn", "batch": 32, "rows": 1, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "length": 511, "ragged": True, "drafts": False},
        # The same batch verifying up to five drafted tokens a sequence.
        {"name": "drafts", "kind": "attn", "batch": 32, "rows": 5, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "length": 509, "ragged": True, "drafts": True},
        # 64 sequences at the end of a 2048-token context: the cache is read
        # at the memory's rate.
        {"name": "long_batch", "kind": "attn", "batch": 64, "rows": 1, "heads": 16, "kv_heads": 16,
         "head_dim": 128, "length": 2040, "ragged": False, "drafts": False},
        # Few sequences of documents, grouped heads: one long axis to split.
        {"name": "documents", "kind": "attn", "batch": 3, "rows": 1, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "length": 100001, "ragged": True, "drafts": False},
        # A serving batch behind one system prompt.
        {"name": "system_prompt", "kind": "prefix", "batch": 32, "rows": 1, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "prefix": 385, "length": 120, "ragged": True,
         "drafts": False},
        # Drafts of many users over one long document.
        {"name": "shared_document", "kind": "prefix", "batch": 64, "rows": 4, "heads": 16,
         "kv_heads": 16, "head_dim": 128, "prefix": 8200, "length": 250, "ragged": True,
         "drafts": True},
        # One user's drafts by a table of n-grams: no draft distribution.
        {"name": "verify_chat", "kind": "verify", "batch": 1, "rows": 4, "vocab": 50257,
         "one_hot": True, "temperature": 0.8, "ragged": False},
        # A serving batch's drafts by a small model.
        {"name": "verify_batch", "kind": "verify", "batch": 32, "rows": 7, "vocab": 50257,
         "one_hot": False, "temperature": 1.0, "ragged": True},
    ]


def _log(rng, low, high):
    """A whole number, uniform in its logarithm."""
    high = max(low, high)
    return min(high, max(low, round(low * (high / low) ** rng.random())))


# (heads, kv_heads, head_dim): the profiles' own, grouped ones, odd head sizes.
_HEADS = [(12, 12, 64), (12, 12, 64), (5, 5, 64), (16, 16, 128), (16, 16, 128), (16, 4, 128),
          (12, 2, 64), (8, 8, 80), (7, 7, 33), (4, 4, 32), (32, 8, 112)]


def draw(rng):
    kind = rng.choice(["cache", "read", "attn", "attn", "attn", "prefix", "prefix", "verify"])
    if kind == "verify":
        rows = rng.randint(1, 8)
        return {"kind": kind, "batch": _log(rng, 1, 256 // (rows + 1)), "rows": rows,
                "vocab": _log(rng, 1000, 50257), "one_hot": rng.random() < 0.4,
                "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5]),
                "ragged": rng.random() < 0.5}
    heads, kv_heads, head_dim = rng.choice(_HEADS)
    shape = {"heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}
    wide = kv_heads * _row_bytes(head_dim)
    if kind in ("cache", "read"):
        batch = _log(rng, 1, 64)
        rows = _log(rng, 1, min(2040, (32 << 20) // (batch * wide)))
        return {"kind": kind, "batch": batch, "rows": rows, **shape,
                "max_rows": rows + _log(rng, 1, 300), "ragged": rng.random() < 0.5}
    batch, rows = _log(rng, 1, 64), rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(9, 24)])
    if kind == "attn":
        if rows * heads // kv_heads > 8:
            batch = min(batch, 16)
        length = _log(rng, rows, min(120000, (190 << 20) // (batch * wide * (1 + rows // 9))))
        return {"kind": kind, "batch": batch, "rows": rows, **shape, "length": length,
                "ragged": rng.random() < 0.5, "drafts": rows > 1 and rng.random() < 0.6}
    rows = min(rows, 6)
    most = max(200, min(40000, (2 << 30) // (batch * rows * heads * _row_bytes(head_dim))))
    return {"kind": kind, "batch": batch, "rows": rows, **shape, "prefix": _log(rng, 33, most),
            "length": _log(rng, rows, 300), "ragged": rng.random() < 0.6,
            "drafts": rows > 1 and rng.random() < 0.6}


# ---- the cache's layout ------------------------------------------------------


def _row_bytes(head_dim):
    return 64 if head_dim <= 64 else 128


def _cap(max_rows):
    return (max_rows + 31) // 32 * 32


def _parts(buffer, slots, kv_heads, max_rows, head_dim):
    """Views of a cache buffer: K codes, V codes, K exponents, V exponents."""
    cap, row = _cap(max_rows), _row_bytes(head_dim)
    n, m = slots * kv_heads * cap * row, slots * kv_heads * cap
    k, v, ke, ve = buffer.split([n, n, m, m])
    return (k.view(slots, kv_heads, cap, row), v.view(slots, kv_heads, cap, row),
            ke.view(slots, kv_heads, cap), ve.view(slots, kv_heads, cap))


def _quantise(x):
    """Codes and exponents of rows x [..., head_dim]: the least power of two
    that takes the row's largest magnitude to 127 or less."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    e = (exponent - 7 + (mantissa > 127 / 128).int()).clamp(min=-126)
    return torch.round(x * _power(-e)[..., None]).to(torch.int8), e.to(torch.int8)


def _power(e):
    """2^e in 32 bits, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _values(codes, exponents, head_dim):
    return codes[..., :head_dim].float() * _power(exponents)[..., None]


def _filled(g, slots, kv_heads, max_rows, head_dim):
    """A cache whose rows hold K and V of N(0, 1) times a factor of each row's
    own between a quarter and four."""
    row, cap = _row_bytes(head_dim), _cap(max_rows)
    buffer = torch.zeros(2 * slots * kv_heads * cap * (row + 1), dtype=torch.int8, device="cuda")
    k, v, ke, ve = _parts(buffer, slots, kv_heads, max_rows, head_dim)
    for codes, exponents in ((k, ke), (v, ve)):
        for s in range(slots):
            x = torch.randn(kv_heads, cap, head_dim, generator=g, device="cuda")
            x *= torch.exp2(4 * torch.rand(kv_heads, cap, 1, generator=g, device="cuda") - 2)
            codes[s, :, :, :head_dim], exponents[s] = _quantise(x)
    return buffer


# ---- inputs ------------------------------------------------------------------


def _spread(case, low, high):
    """One whole number of [low, high] per sequence, the same for every seed:
    uneven ones where the case is ragged, `high` otherwise."""
    b = case["batch"]
    if not case["ragged"]:
        return torch.full((b,), high, dtype=torch.int32)
    return torch.tensor([high - (i * 7919) % (high - low + 1) for i in range(b)],
                        dtype=torch.int32)


def _counts(case):
    """New rows of each sequence: of drafts, from none up to all."""
    r, b = case["rows"], case["batch"]
    if not case["drafts"]:
        return torch.full((b,), r, dtype=torch.int32)
    return torch.tensor([r - (i * 5) % (r + 1) for i in range(b)], dtype=torch.int32)


def _verify_inputs(case, g):
    """Target logits N(0, 2.5^2) plus a few likely ids, the draft's logits
    near them, and drafts drawn from the draft's distribution (one-hot drafts:
    from the target's own)."""
    b, r, n = case["batch"], case["rows"], case["vocab"]
    target = torch.randn(b, r + 1, n, generator=g, device="cuda") * 2.5
    likely = torch.randint(0, n, (b, r + 1, 8), generator=g, device="cuda")
    target.scatter_add_(-1, likely, torch.full(likely.shape, 8.0, device="cuda"))
    draft = None
    near = target[:, :r]
    if not case["one_hot"]:
        draft = target[:, :r] + torch.randn(b, r, n, generator=g, device="cuda") * 0.7
        near = draft
    t = case["temperature"] if case["temperature"] > 0 else 0.3
    noise = torch.rand(b, r, n, generator=g, device="cuda").clamp_(min=1e-7)
    tokens = (near / t - torch.log(-torch.log(noise))).argmax(-1).int()
    uniforms = torch.rand(b, r + 1, generator=g, device="cuda", dtype=torch.float64)
    return target, draft, tokens, uniforms


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = {"case": case}
    if kind == "verify":
        target, draft, tokens, uniforms = _verify_inputs(case, g)
        state |= {"target": target, "draft": draft, "tokens": tokens, "uniforms": uniforms,
                  "counts": _spread(case, 0, case["rows"]).cuda()}
        return state
    b, kh, hd = case["batch"], case["kv_heads"], case["head_dim"]
    if kind in ("cache", "read"):
        rows, most = case["rows"], case["max_rows"]
        counts = _spread(case, max(0, rows // 3), rows)
        state["counts"] = counts.cuda()
        state["pos"] = ((torch.arange(b, dtype=torch.int32) * 31) % (most - rows + 1)).cuda()
        if kind == "cache":
            qkv = torch.randn(b * rows, (case["heads"] + 2 * kh) * hd, generator=g, device="cuda")
            state["qkv"] = qkv
            size = 2 * b * kh * _cap(most) * (_row_bytes(hd) + 1)
            state["cache"] = torch.zeros(size, dtype=torch.int8, device="cuda")
        else:
            state["cache"] = _filled(g, b, kh, most, hd)
        return state
    counts = _counts(case)
    ends = torch.maximum(_spread(case, max(1, case["length"] // 4), case["length"]), counts)
    state["counts"], state["pos"] = counts.cuda(), (ends - counts).cuda()
    state["cache"] = _filled(g, b, kh, case["length"], hd)
    state["q"] = torch.randn(b, case["rows"], case["heads"], hd, generator=g, device="cuda")
    if kind == "prefix":
        state["prefix"] = _filled(g, 1, kh, case["prefix"], hd)
        state["prefix_len"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
    return state


# ---- one pass ----------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _own_pass(state)
    if case["kind"] == "cache":
        return _plain_cache(state)
    if case["kind"] == "read":
        return _plain_read(state)
    if case["kind"] == "verify":
        return _plain_verify(state)
    return _plain_attention(state)


def _kv_rows(state):
    """The K and V columns of the fused projection, [batch, rows, kv_heads,
    head_dim] each: after the heads' Q come kv_heads of K, then of V."""
    c = state["case"]
    q, kv = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    shape = (c["batch"], c["rows"], c["kv_heads"], c["head_dim"])
    return (state["qkv"][:, q:q + kv].reshape(shape),
            state["qkv"][:, q + kv:q + 2 * kv].reshape(shape))


def _live(state):
    """[batch, rows]: which of the case's rows a sequence has."""
    t = torch.arange(state["case"]["rows"], device="cuda")
    return t < state["counts"][:, None]


def _at(state):
    """Each sequence's and row's place in the cache, [batch, rows] twice."""
    c = state["case"]
    t = torch.arange(c["rows"], device="cuda")
    place = state["pos"][:, None].long() + t
    return torch.arange(c["batch"], device="cuda")[:, None].expand_as(place), place


def _plain_cache(state):
    c = state["case"]
    parts = _parts(state["cache"], c["batch"], c["kv_heads"], c["max_rows"], c["head_dim"])
    live = _live(state)[..., None]
    b, at = _at(state)
    for rows, codes, exponents in zip(_kv_rows(state), parts[:2], parts[2:]):
        codes, exponents = codes.transpose(1, 2)[..., :c["head_dim"]], exponents.transpose(1, 2)
        q, e = _quantise(rows)
        codes[b, at] = torch.where(live[..., None], q, codes[b, at])
        exponents[b, at] = torch.where(live, e, exponents[b, at])
    return _plain_read(state)


def _plain_read(state):
    c = state["case"]
    k, v, ke, ve = _parts(state["cache"], c["batch"], c["kv_heads"], c["max_rows"], c["head_dim"])
    live = _live(state)[..., None, None]
    b, at = _at(state)
    out = {}
    for name, codes, exponents in (("k", k, ke), ("v", v, ve)):
        x = _values(codes.transpose(1, 2)[b, at], exponents.transpose(1, 2)[b, at], c["head_dim"])
        out[name] = torch.where(live, x, torch.zeros_like(x))
    return out


def _plain_attention(state):
    c = state["case"]
    b, t, h, kh, hd = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    k, v, ke, ve = _parts(state["cache"], b, kh, c["length"], hd)
    k, v = _values(k, ke, hd), _values(v, ve, hd)
    cap = k.shape[2]
    # Rows [batch, kv_heads, group * rows, head_dim].
    q = state["q"].view(b, t, kh, h // kh, hd).permute(0, 2, 3, 1, 4).reshape(b, kh, -1, hd)
    score = torch.matmul(q, k.transpose(-1, -2)) * hd ** -0.5
    last = state["pos"][:, None] + torch.arange(t, device="cuda")
    last = torch.where(_live(state), last, -1).repeat(1, h // kh)[:, None, :, None]
    seen = torch.arange(cap, device="cuda") <= last
    score = score.masked_fill(~seen, float("-inf"))
    if c["kind"] == "prefix":
        pk, pv, pke, pve = _parts(state["prefix"], 1, kh, c["prefix"], hd)
        pk, pv = _values(pk, pke, hd)[0], _values(pv, pve, hd)[0]
        n = pk.shape[1]
        every = q.transpose(0, 1).reshape(kh, -1, hd)
        first = torch.matmul(every, pk.transpose(-1, -2)) * hd ** -0.5
        first = first.view(kh, b, -1, n).transpose(0, 1)
        there = (torch.arange(n, device="cuda") < state["prefix_len"]) & (last >= 0)
        score = torch.cat([first.masked_fill(~there, float("-inf")), score], -1)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if c["kind"] == "prefix":
        head = p[..., :n].transpose(0, 1).reshape(kh, -1, n)
        x = torch.matmul(head, pv).view(kh, b, -1, hd).transpose(0, 1)
        x = x + torch.matmul(p[..., n:], v)
    else:
        x = torch.matmul(p, v)
    x = torch.where(total > 0, x / total, torch.zeros_like(x))
    lse = (top + torch.log(total))[..., 0]
    order = (0, 3, 1, 2)
    return {"out": x.view(b, kh, h // kh, t, hd).permute(*order, 4).reshape(b, t, h, hd),
            "lse": lse.view(b, kh, h // kh, t).permute(order).reshape(b, t, h)}


def _plain_verify(state):
    c = state["case"]
    b, r, n = c["batch"], c["rows"], c["vocab"]
    target, tokens, counts = state["target"], state["tokens"].long(), state["counts"].long()
    live = _live(state)
    if c["temperature"] <= 0:
        best = target.argmax(-1)
        accept = (tokens == best[:, :r]) & live
        chance = accept.float()
        taken = accept.int().cumprod(-1).sum(-1)
        last = best.gather(1, taken[:, None])[:, 0]
    else:
        p = _softmax64(target, c["temperature"])
        q = torch.zeros_like(p[:, :r]).scatter_(-1, tokens[..., None], 1.0) if c["one_hot"] \
            else _softmax64(state["draft"], c["temperature"])
        px, qx = (x.gather(-1, tokens[..., None])[..., 0] for x in (p[:, :r], q))
        chance = torch.where(live, (px / qx).clamp(max=1.0), 0.0).float()
        accept = (state["uniforms"][:, :r] * qx < px) & live
        taken = accept.int().cumprod(-1).sum(-1)
        rows = torch.arange(b, device="cuda")
        weight = p[rows, taken]
        less = q[rows, taken.clamp(max=r - 1)]
        rest = (weight - less).clamp(min=0.0)
        cut = (taken < counts) & (rest.sum(-1) > 0)
        cdf = torch.where(cut[:, None], rest, weight).cumsum(-1)
        point = state["uniforms"][:, r:] * cdf[:, -1:]
        last = (cdf <= point).sum(-1).clamp(max=n - 1)
    place = torch.arange(r + 1, device="cuda")
    out = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(place < taken[:, None], out, -1)
    out = torch.where(place == taken[:, None], last[:, None], out)
    return {"tokens": out.int(), "counts": (taken + 1).int(), "chance": chance}


def _softmax64(x, temperature):
    x = x.double()
    p = torch.exp((x - x.amax(-1, keepdim=True)) / temperature)
    return p / p.sum(-1, keepdim=True)


def _pointer(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _plan(state):
    """What a program keeps beside its buffers: the backend, the cache
    handles, the call's sizes, its outputs and workspace."""
    global _backend
    hip = importlib.import_module("akasha-core_amd").hip
    if _backend is None:
        _backend = hip.Backend(0)
    c, kind = state["case"], state["case"]["kind"]
    empty = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
    p = {name: _pointer(t) for name, t in state.items() if isinstance(t, torch.Tensor)}
    b, r = c["batch"], c["rows"]
    if kind == "verify":
        p["out"] = {"tokens": empty(b, r + 1, dtype=torch.int32),
                    "counts": empty(b, dtype=torch.int32), "chance": empty(b, r)}
        p["size"] = hip.verify_drafts_workspace(b, r, c["vocab"])
        p["work"] = empty(max(1, p["size"]), dtype=torch.int8)
        return p
    kh, hd = c["kv_heads"], c["head_dim"]
    p["q8"] = hip.Q8Cache(_backend, b, c.get("length") or c["max_rows"], kh, hd, p["cache"])
    if kind in ("cache", "read"):
        p["out"] = {"k": empty(b, r, kh, hd), "v": empty(b, r, kh, hd)}
        if kind == "cache":
            at = 4 * c["heads"] * hd
            p["k"] = ctypes.c_void_p(state["qkv"].data_ptr() + at)
            p["v"] = ctypes.c_void_p(state["qkv"].data_ptr() + at + 4 * kh * hd)
        return p
    width = c["heads"] * hd
    p["shape"] = hip.AttnQ8(b, r, c["heads"], width, width, hd ** -0.5, c["length"])
    p["out"] = {"out": empty(b, r, c["heads"], hd), "lse": empty(b, r, c["heads"])}
    p["pre"] = hip.Q8Cache(_backend, 1, c["prefix"], kh, hd, p["prefix"]) \
        if kind == "prefix" else None
    p["size"] = hip.attn_q8_workspace(p["shape"], p["q8"], p["pre"])
    p["work"] = empty(max(1, p["size"]), dtype=torch.int8)
    return p


def _own_pass(state):
    c, kind = state["case"], state["case"]["kind"]
    if "plan" not in state:
        state["plan"] = _plan(state)
        torch.cuda.synchronize()
    p = state["plan"]
    out, b, r = p["out"], c["batch"], c["rows"]
    if kind == "verify":
        _backend.verify_drafts(p["target"], p.get("draft"), p["tokens"], b, r, c["vocab"],
                               _pointer(out["tokens"]), _pointer(out["counts"]),
                               _pointer(out["chance"]), temperature=c["temperature"],
                               counts=p["counts"], uniforms=p["uniforms"],
                               workspace=_pointer(p["work"]), workspace_bytes=p["size"])
        return out
    if kind in ("cache", "read"):
        if kind == "cache":
            _backend.cache_write_q8(p["k"], p["v"], p["q8"], b, r,
                                    (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"], p["pos"],
                                    p["counts"])
        _backend.cache_read_q8(p["q8"], _pointer(out["k"]), _pointer(out["v"]), b, r,
                               c["kv_heads"] * c["head_dim"], p["pos"], p["counts"])
        return out
    if kind == "attn":
        _backend.attn_cached_q8(p["q"], p["q8"], _pointer(out["out"]), _pointer(out["lse"]),
                                p["shape"], p["pos"], p["counts"], workspace=_pointer(p["work"]),
                                workspace_bytes=p["size"])
        return out
    _backend.attn_prefix_q8(p["q"], p["pre"], p["prefix_len"], p["q8"], _pointer(out["out"]),
                            _pointer(out["lse"]), p["shape"], p["pos"], p["counts"],
                            workspace=_pointer(p["work"]), workspace_bytes=p["size"])
    return out


# ---- what a pass cannot do without -------------------------------------------


def work(case):
    """Each input of the live rows read once, each output written once; an
    element of the cache is a byte, its row's exponent another."""
    b, r = case["batch"], case["rows"]
    if case["kind"] == "verify":
        live = int((_spread(case, 0, r)).sum())
        logits = (live + b + (0 if case["one_hot"] or case["temperature"] <= 0 else live))
        return {"bytes": 4 * logits * case["vocab"] + b * (r + 1) * 12 + b * r * 8 + b * 8,
                "flops": 3 * logits * case["vocab"]}
    h, kh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] in ("cache", "read"):
        live = int(_spread(case, max(0, r // 3), r).sum())
        values, held = 2 * 4 * kh * hd, 2 * kh * (hd + 1)
        if case["kind"] == "read":
            return {"bytes": live * held + b * r * values, "flops": 2 * live * kh * hd}
        return {"bytes": live * (values + 2 * held) + b * r * values, "flops": 8 * live * kh * hd}
    counts = _counts(case)
    ends = torch.maximum(_spread(case, max(1, case["length"] // 4), case["length"]), counts)
    read = int(ends[counts > 0].sum())
    pairs = sum(n * e - n * (n - 1) // 2 for n, e in zip(counts.tolist(), ends.tolist()))
    if case["kind"] == "prefix":
        read += case["prefix"]
        pairs += case["prefix"] * int(counts.sum())
    return {"bytes": 2 * read * kh * (hd + 1) + 4 * int(counts.sum()) * h * hd
            + 4 * b * r * h * (hd + 1), "flops": 4 * pairs * h * hd}


# ---- 64 bits -----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "verify":
        return {"tokens": None, "counts": None, "chance": _exact_chance(s)}
    b, r, kh, hd = case["batch"], case["rows"], case["kv_heads"], case["head_dim"]
    pos, counts = s["pos"].tolist(), s["counts"].tolist()
    if kind in ("cache", "read"):
        out = torch.zeros(2, b, r, kh, hd, dtype=torch.float64, device="cuda")
        for i in range(b):
            n = counts[i]
            if kind == "read":
                for which in range(2):
                    x = _held64(s["cache"], b, kh, case["max_rows"], hd, i, which)
                    out[which, i, :n] = x[:, pos[i]:pos[i] + n].transpose(0, 1)
                continue
            rows = s["qkv"].view(b, r, -1)[i, :n, case["heads"] * hd:].double()
            for which in range(2):
                x = rows[:, which * kh * hd:(which + 1) * kh * hd].reshape(n, kh, hd)
                # The least step 2^e with the largest magnitude within 127 steps.
                e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 127))
                out[which, i, :n] = torch.round(x / 2.0 ** e) * 2.0 ** e
        return {"k": out[0], "v": out[1]}
    h = case["heads"]
    out = torch.zeros(b, r, h, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((b, r, h), float("-inf"), dtype=torch.float64, device="cuda")
    ahead = 0
    if kind == "prefix":
        ahead = case["prefix"]
        pre = [_held64(s["prefix"], 1, kh, ahead, hd, 0, w)[:, :ahead] for w in range(2)]
    for i in range(b):
        n = counts[i]
        if not n:
            continue
        end = pos[i] + n
        k, v = (_held64(s["cache"], b, kh, case["length"], hd, i, w)[:, :end] for w in range(2))
        if ahead:
            k, v = torch.cat([pre[0], k], 1), torch.cat([pre[1], v], 1)
        for j in range(n):
            m = ahead + pos[i] + j + 1
            q = s["q"][i, j].double().view(kh, h // kh, hd)
            x = torch.matmul(q, k[:, :m].transpose(1, 2).contiguous()) / hd ** 0.5
            lse[i, j] = torch.logsumexp(x, -1).view(h)
            out[i, j] = torch.matmul(torch.softmax(x, -1), v[:, :m]).view(h, hd)
    return {"out": out, "lse": lse}


def _held64(buffer, slots, kv_heads, max_rows, head_dim, slot, which):
    """What slot `slot` of a cache holds for K (0) or V (1): [kv_heads, cap, head_dim]."""
    row, cap = (64 if head_dim <= 64 else 128), -(-max_rows // 32) * 32
    heads = slots * kv_heads * cap
    at = (which * slots + slot) * kv_heads * cap
    codes = buffer[at * row:(at + kv_heads * cap) * row].view(kv_heads, cap, row)
    at += 2 * heads * row
    e = buffer[at:at + kv_heads * cap].view(kv_heads, cap, 1)
    return codes[:, :, :head_dim].double() * 2.0 ** e.double()


def _exact_chance(s):
    c = s["case"]
    r = c["rows"]
    live = np.arange(r) < s["counts"].cpu().numpy()[:, None]
    tokens = s["tokens"].long()[..., None]
    if c["temperature"] <= 0:
        x = s["target"][:, :r]
        first = (x == x.max(-1, keepdim=True).values).int().argmax(-1)
        return (first == tokens[..., 0]).double() * torch.from_numpy(live).cuda()
    logp = (s["target"][:, :r].double() / c["temperature"]).log_softmax(-1).gather(-1, tokens)
    if not c["one_hot"]:
        logp = logp - (s["draft"].double() / c["temperature"]).log_softmax(-1).gather(-1, tokens)
    return logp[..., 0].exp().clamp(max=1.0) * torch.from_numpy(live).cuda()
