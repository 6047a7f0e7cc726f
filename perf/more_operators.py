"""Operators around the paged key-value cache, as they are timed: one pass each of

* ``decode``  attention of one new token per sequence, where groups of sequences share their first tokens: those
              are read once for the whole group (answers forked from one document);
* ``prompt``  the same for several new tokens per sequence (questions on one document), causal;
* ``append``  new queries, keys and values of a joint product: norm of each head, rotary positions, keys and values
              into the pages of their sequences, queries returned;
* ``rotary``  rotary positions alone, and their gradient.

Shapes: K and V [layers][pages][kv_heads][page][dim], table [sequences][width] page numbers (-1: no page), lengths
[sequences]; group g has the sequences groups[g] .. groups[g + 1] - 1, which share their first shared[g] tokens, read
through the table's row of its first sequence.  ``own`` False: elementary torch operations in 32 bits, angles in 64.
``own`` True: the calls of ``bfvgpu.PagedKv`` and ``bfvgpu.Rotary``.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------ cases
def _case(name, op, **kw):
    c = dict(op=op, q_heads=16, kv_heads=8, dim=128, page=16, dtype="bf16", layout="hnd")
    if op in ("decode", "prompt"):
        c.update(seqs=1, groups=1, prefix=512, own=16, new=1, even=False)
    else:
        c.update(source="bf16", rotated=128, style="half", base=1e6, scaling="none", factor=1.0, norm=False)
        if op == "append":
            c.update(seqs=1, length=512, new=1, ragged=False, queries=True)
        else:
            c.update(tokens=1, far=4096, inverse=False)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # sixteen answers forked from one 1000-token document (62 full pages are shared), a few tokens each; latency
        _case("shared answers", "decode", seqs=16, prefix=992, own=32),
        # a serving batch: four system prompts or documents, sessions at mixed lengths
        _case("shared batch", "decode", seqs=64, groups=4, prefix=4096, own=512),
        # many sessions on one long document, few key heads
        _case("shared long", "decode", seqs=128, prefix=65536, own=1024, q_heads=32, kv_heads=4, page=64, dtype="fp16"),
        # sixteen questions on one document, none longer than 64 tokens
        _case("shared questions", "prompt", seqs=16, prefix=4096, own=64, new=64),
        # chunks of six sessions on two documents: three query heads per key head, pages with the heads inside
        _case("shared chunks", "prompt", seqs=6, groups=2, prefix=8192, own=2048, new=1024, q_heads=12, kv_heads=4, dim=64,
              page=32, dtype="fp16", layout="nhd"),
        # one decode step of 64 sequences: head norms, rotation, keys and values into their pages, queries out; latency
        _case("rotated step", "append", seqs=64, length=4096, ragged=True, norm=True),
        # prompts whose projections come in 32 bits, positions scaled for four times the trained length
        _case("rotated prompts", "append", seqs=8, length=4096, new=4096, ragged=True, norm=True, source="f32", scaling="yarn",
              factor=4.0),
        # half of each head rotated, in pairs of neighbours, at far positions of a long document
        _case("rotated chunk", "append", length=131071, new=8191, q_heads=32, kv_heads=4, page=64, dtype="fp16", source="fp16",
              layout="nhd", rotated=64, style="interleaved", base=1e4),
        # the queries and keys of one decode step of 16 sequences; latency
        _case("rotary step", "rotary", tokens=16, q_heads=24, far=131071),
        # a prompt's queries, with head norms
        _case("rotary prompt", "rotary", tokens=16384, q_heads=32, far=16384, norm=True),
        # the gradient of a rotation of a quarter of each head
        _case("rotary gradient", "rotary", tokens=8191, q_heads=12, dim=96, rotated=24, dtype="f32", source="f32", far=8191,
              inverse=True, scaling="linear", factor=2.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    largest = {}
    for c in listed():
        w = work(c)
        m = largest.setdefault(c["op"], [0, 0, 0])
        largest[c["op"]] = [max(m[0], w["bytes"]), max(m[1], w["flops"]), max(m[2], _padded(c))]
    while True:
        op = rng.choice(["decode", "decode", "prompt", "prompt", "append", "append", "rotary"])
        kv = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 72, 96, 128, 128])
        c = _case(None, op, kv_heads=kv, q_heads=kv * rng.choice([1, 2, 3, 4, 5, 8]), dim=dim, page=rng.choice([16, 32, 64, 128]),
                  dtype=rng.choice(["bf16", "fp16"]), layout=rng.choice(["hnd", "nhd"]))
        if op in ("decode", "prompt"):
            c.update(seqs=_log(rng, 1, 128 if op == "decode" else 32), prefix=_log(rng, 1, 65536 if op == "decode" else 16384),
                     own=_log(rng, 1, 1024 if op == "decode" else 4096), even=rng.random() < 0.3)
            c["groups"] = _log(rng, 1, min(8, c["seqs"]))
            if op == "prompt":
                c["new"] = c["own"] if rng.random() < 0.5 else _log(rng, 1, c["own"])
        else:
            c.update(rotated=dim if rng.random() < 0.5 else 4 * rng.randint(1, dim // 4), style=rng.choice(["half", "interleaved"]),
                     base=rng.choice([1e4, 5e5, 1e6]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]), norm=rng.random() < 0.5)
            if c["rotated"] < 8 and c["scaling"] in ("ntk", "yarn"):
                c["scaling"] = "none"
            c["factor"] = 1.0 if c["scaling"] == "none" else rng.choice([2.0, 4.0, 7.5])
            if op == "append":
                c.update(seqs=_log(rng, 1, 128), length=_log(rng, 1, 131071), ragged=rng.random() < 0.7,
                         queries=rng.random() < 0.8)
                c["new"] = 1 if rng.random() < 0.4 else _log(rng, 1, min(8192, c["length"]))
                c["source"] = rng.choice([c["dtype"], "f32"])
            else:
                c.update(tokens=_log(rng, 1, 16384), far=_log(rng, 1, 131071), inverse=rng.random() < 0.4)
                c["dtype"] = rng.choice([c["dtype"], "f32"])
                c["source"] = c["dtype"]
                c["norm"] = c["norm"] and not c["inverse"]
        w, (b, f, g) = work(c), largest[op]
        if w["bytes"] <= b and w["flops"] <= f and _padded(c) <= g:
            return c


def _sizes(case):
    """The sizes of a case, the same for every seed: (groups, shared, [(length, new tokens)])."""
    if case["op"] == "append":
        rng = random.Random("%(op)s %(seqs)d %(length)d %(new)d" % case)
        out = []
        for s in range(case["seqs"]):
            if not case["ragged"] or s == 0:
                out.append((case["length"], case["new"]))
            elif case["new"] == case["length"]:
                n = rng.randint(1, case["length"])
                out.append((n, n))
            else:
                n = rng.randint(1, case["length"])
                out.append((n, min(n, rng.randint(1, case["new"]))))
        return None, None, out
    rng = random.Random("%(op)s %(seqs)d %(groups)d %(prefix)d %(own)d %(new)d" % case)
    cuts = sorted(rng.sample(range(1, case["seqs"]), case["groups"] - 1))
    groups = [0] + cuts + [case["seqs"]]
    shared = [case["prefix"]] + [rng.randint(1, case["prefix"]) for _ in range(case["groups"] - 1)]
    lens, g = [], 0
    for s in range(case["seqs"]):
        g += s == groups[g + 1]
        mine = case["own"] if s == 0 or case["even"] else rng.randint(1, case["own"])
        new = min(mine, case["new"] if s == 0 or case["even"] or case["new"] == case["own"] else rng.randint(1, case["new"]))
        lens.append((shared[g] + mine, new))
    return groups, shared, lens


def _padded(case):
    """Size of the padded arrays of the plain form."""
    if case["op"] == "rotary":
        return 0
    groups, shared, lens = _sizes(case)
    if case["op"] == "append":
        return sum(-(-n // case["page"]) for n, _ in lens) * case["page"] * case["kv_heads"] * case["dim"]
    new = [n for _, n in lens]
    most = max(sum(new[a:b]) for a, b in zip(groups, groups[1:]))
    rows = case["groups"] * most * max(shared) + case["seqs"] * max(new) * case["own"]
    return max(case["q_heads"] * rows, case["seqs"] * (case["own"] + 2 * case["page"]) * case["kv_heads"] * case["dim"])


def work(case):
    h, g, d = case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n = case["tokens"] * h
        return {"bytes": 2 * n * d * BYTES[case["dtype"]] + 4 * case["tokens"], "flops": n * (3 * case["rotated"] + (3 * d if case["norm"] else 0))}
    groups, shared, lens = _sizes(case)
    tokens = sum(n for _, n in lens)
    if case["op"] == "append":
        rows = (h if case["queries"] else 0) + g
        return {"bytes": tokens * (rows + g) * d * (BYTES[case["source"]] + 2) + 4 * 3 * case["seqs"],
                "flops": tokens * rows * (3 * case["rotated"] + (3 * d if case["norm"] else 0))}
    first = [shared[i] for i, (a, b) in enumerate(zip(groups, groups[1:])) for _ in range(a, b)]
    keys = sum(shared) + sum(n - p for (n, _), p in zip(lens, first))
    pairs = sum(n * (n + 1) // 2 - (n - new) * (n - new + 1) // 2 for n, new in lens)
    return {"bytes": 2 * 2 * keys * g * d + 2 * 2 * tokens * h * d, "flops": 4 * pairs * h * d}


# ----------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    h, g, d, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    state = {k: case[k] for k in ("op", "page", "style", "base", "scaling", "factor", "rotated", "inverse") if k in case}
    state["scale"] = 1.0 / math.sqrt(d)
    if op in ("append", "rotary"):
        for name in ("q_norm", "k_norm"):
            w = 1 + 0.2 * torch.randn(d, device=dev, generator=gen)
            state[name] = w if case["norm"] else None
    if op == "rotary":
        n = case["tokens"]
        # prompts that start anywhere below `far`
        at = torch.randint(0, case["far"], (), device=dev, generator=gen)
        state["positions"] = ((torch.arange(n, device=dev) + at) % case["far"]).to(torch.int32)
        state["x"] = torch.randn(n, h * d, device=dev, generator=gen, dtype=torch.float32).to(dt).unflatten(1, (h, d))
        return state
    groups, shared, lens = _sizes(case)
    firsts = [0] * case["seqs"]  # pages that a sequence has of its group
    if op != "append":
        for a, b, p in zip(groups, groups[1:], shared):
            firsts[a:b] = [0] + [p // page] * (b - a - 1)
    counts = [-(-n // page) for n, _ in lens]
    used = sum(c - f for c, f in zip(counts, firsts))
    total = used + 3
    wide = torch.float32 if op == "append" else dt
    rand = lambda *s: torch.randn(*s, device=dev, generator=gen, dtype=wide)  # noqa: E731
    shape = (1, total, g, page, d) if case["layout"] == "hnd" else (1, total, page, g, d)
    k, v = (torch.randn(*shape, device=dev, generator=gen, dtype=dt) for _ in range(2))
    if case["layout"] == "nhd":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    # pages in the order of a cache that has been in use: any page may hold any part
    perm = torch.randperm(total, device=dev, generator=gen).to(torch.int32)
    width = max(counts) + 1
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=dev)
    at, firsts_, counts_ = torch.arange(width, device=dev), ints(firsts)[:, None], ints(counts)[:, None]
    table[(at >= firsts_) & (at < counts_)] = perm[:used]
    if op != "append":
        for a, b, p in zip(groups, groups[1:], shared):
            if b - a > 1 and p >= page:
                table[a + 1:b, :p // page] = table[a, :p // page]
        state.update(groups=ints(groups), shared=ints(shared), prefix_pages=-(-max(shared) // page),
                     own_pages=max(c - p // page for c, p in zip(counts, (shared[i] for i, (a, b) in enumerate(zip(groups, groups[1:])) for _ in range(a, b)))),
                     most_of_group=max(sum(n for _, n in lens[a:b]) for a, b in zip(groups, groups[1:])))
    new = [n for _, n in lens]
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    state.update(k=k, v=v, table=table, lengths=ints([n for n, _ in lens]), starts=ints(starts), most=max(new),
                 single=max(new) == 1)
    # queries, keys and values lie in the rows of a joint q/k/v product, as the layer's call leaves them
    row = rand(starts[-1], (h + 2 * g) * d)
    if op == "append":
        row = row.to(DTYPES[case["source"]])
        state["k_new"] = row[:, h * d:(h + g) * d].unflatten(1, (g, d))
        state["v_new"] = row[:, (h + g) * d:].unflatten(1, (g, d))
    state["q"] = row[:, :h * d].unflatten(1, (h, d)) if op != "append" or case["queries"] else None
    return state


# ------------------------------------------------------------------------------------------- plain forms
def _frequencies(s, dev):
    """Angle per position of each pair in 64 bits, and the factor of the rotated values."""
    n, base, f = s["rotated"], s["base"], s["factor"]
    i = torch.arange(0, n, 2, dtype=torch.float64, device=dev)
    if s["scaling"] == "ntk":
        base = base * f ** (n / (n - 2))
    w = base ** (-i / n)
    if s["scaling"] == "linear":
        return w / f, 1.0
    if s["scaling"] != "yarn":
        return w, 1.0
    # full turns over the trained length: at least 32 keep their frequency, at most one is divided by the factor
    turn = lambda turns: n * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(turn(32)), 0), min(math.ceil(turn(1)), n - 1)
    ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
    return w * (1 - ramp) + w / f * ramp, 0.1 * math.log(f) + 1


def _rotate(s, x, positions, norm):
    """x [tokens][heads][dim] in 32 bits: norm of each head, then the rotation."""
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * norm
    w, factor = _frequencies(s, x.device)
    angle = positions.double()[:, None] * w
    cos, sin = ((f(angle) * factor).float()[:, None] for f in (torch.cos, torch.sin))
    if s.get("inverse"):
        sin = -sin
    n = s["rotated"]
    y = x.clone()
    if s["style"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2], y[..., n // 2:n] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :n:2], x[..., 1:n:2]
        y[..., :n:2], y[..., 1:n:2] = a * cos - b * sin, b * cos + a * sin
    return y


def _sequence_of(starts, tokens):
    t = torch.arange(tokens, device=starts.device)
    seq = torch.searchsorted(starts[1:].long(), t, right=True)
    return seq, t - starts.long()[seq]


def _part(q, k, v, seen, scale):
    """q [B][G][R][rows][D], k, v [B][G][T][D], seen [B][rows or 1][T]: (maximum, sum, weighted values) of the seen keys."""
    b, g, r, n, d = q.shape
    x = (q.reshape(b, g, r * n, d) @ k.transpose(2, 3)) * scale
    x = x.view(b, g, r, n, -1).masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.clamp(min=-3e38))
    return m, p.sum(-1, keepdim=True), (p.flatten(2, 3) @ v).view(b, g, r, n, d)


def _plain_shared(s):
    q, page, table, lengths = s["q"].float(), s["page"], s["table"].clamp(min=0).long(), s["lengths"].long()
    groups, shared = s["groups"].long(), s["shared"].long()
    tokens, h, d = q.shape
    pages = lambda x, at: x[0][at].transpose(1, 2).flatten(2, 3).float()  # noqa: E731
    seq, i = _sequence_of(s["starts"], tokens)
    group_of = torch.searchsorted(groups[1:], torch.arange(len(lengths), device=q.device), right=True)
    starts = s["starts"].long()
    g, r = s["k"].shape[2], h // s["k"].shape[2]

    def rows(batch, at, n):  # tokens as padded rows [batch][key head][query head of it][rows][dim]
        x = q.new_zeros(batch, n, h, d)
        x[at] = q
        return x.view(batch, n, g, r, d).permute(0, 2, 3, 1, 4)

    def back(x, at):  # and back: [tokens][heads][...]
        return x.permute(0, 3, 1, 2, 4)[at].reshape(tokens, h, -1)

    # the shared tokens, all rows of a group at once
    at = (group_of[seq], torch.arange(tokens, device=q.device) - starts[groups[:-1]][group_of[seq]])
    first = table[groups[:-1], :s["prefix_pages"]]
    j = torch.arange(first.shape[1] * page, device=q.device)
    prefix = _part(rows(len(shared), at, s["most_of_group"]), pages(s["k"], first), pages(s["v"], first),
                   (j < shared[:, None])[:, None], s["scale"])
    m0, l0, o0 = (back(x, at) for x in prefix)
    # each sequence's own
    begin = shared[group_of] // page
    slots = begin[:, None] + torch.arange(s["own_pages"], device=q.device)
    mine = table.gather(1, slots.clamp(max=table.shape[1] - 1))
    j = begin[:, None] * page + torch.arange(s["own_pages"] * page, device=q.device)
    new = starts[1:] - starts[:-1]
    pos = (lengths - new)[:, None] + torch.arange(s["most"], device=q.device)
    seen = (j[:, None] <= pos[:, :, None]) & (j >= shared[group_of][:, None])[:, None]
    part = _part(rows(len(lengths), (seq, i), s["most"]), pages(s["k"], mine), pages(s["v"], mine), seen, s["scale"])
    m1, l1, o1 = (back(x, (seq, i)) for x in part)
    m = torch.maximum(m0, m1).clamp(min=-3e38)
    f0, f1 = torch.exp(m0 - m), torch.exp(m1 - m)
    total = f0 * l0 + f1 * l1
    return ((f0 * o0 + f1 * o1) / torch.where(total > 0, total, 1.0)).to(s["q"].dtype)


def _plain(s):
    if s["op"] == "rotary":
        return _rotate(s, s["x"].float(), s["positions"], s["q_norm"]).to(s["x"].dtype)
    if s["op"] != "append":
        return _plain_shared(s)
    k, v, page = s["k"][0], s["v"][0], s["page"]
    seq, i = _sequence_of(s["starts"], s["k_new"].shape[0])
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    pos = (s["lengths"].long() - new)[seq] + i
    at = s["table"][seq, pos // page].long()
    k[at, :, pos % page] = _rotate(s, s["k_new"].float(), pos, s["k_norm"]).to(k.dtype)
    v[at, :, pos % page] = s["v_new"].to(v.dtype)
    if s["q"] is None:
        return s["k"], s["v"]
    return s["k"], s["v"], _rotate(s, s["q"].float(), pos, s["q_norm"]).to(k.dtype)


# --------------------------------------------------------------------------------- the framework's calls
_kept = {}


def _held(s):
    """The cache and the rotation that a program holds for as long as it holds its pages."""
    if "held" not in s:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "privacy-rag_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import bfvgpu
        if "ctx" not in _kept:  # the small transform context: n = 4096, 36/36/37-bit primes
            _kept["ctx"] = bfvgpu.Context(4096, bfvgpu.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=0)
        cache = bfvgpu.PagedKv(_kept["ctx"], s["k"], s["v"]) if "k" in s else None
        rotary = None
        if "style" in s:
            rotary = bfvgpu.Rotary(_kept["ctx"], s["rotated"], base=s["base"], layout=s["style"], scaling=s["scaling"],
                                   factor=s["factor"], trained=4096)
        s["held"] = cache, rotary
    return s["held"]


def run(state):
    if not own:
        return _plain(state)
    s = state
    cache, rotary = _held(s)
    if s["op"] == "rotary":
        return rotary.apply(s["x"], s["positions"], norm=s["q_norm"], inverse=s["inverse"])
    if s["op"] == "append":
        starts = None if s["single"] else s["starts"]
        q = cache.append_rotary(s["k_new"], s["v_new"], rotary, starts, s["table"], s["lengths"], q=s["q"], q_norm=s["q_norm"],
                                k_norm=s["k_norm"])
        return (s["k"], s["v"]) if q is None else (s["k"], s["v"], q)
    if s["op"] == "decode":
        return cache.decode_shared(s["q"], s["table"], s["lengths"], s["groups"], s["shared"], scale=s["scale"])
    return cache.prompt_shared(s["q"], s["starts"], s["table"], s["lengths"], s["groups"], s["shared"], scale=s["scale"])


# --------------------------------------------------------------------------------- the definition in 64 bits
def _turned(case, x, positions, weight):
    """One tensor [tokens][heads][dim] in 64 bits, pair by pair."""
    x = x.double()
    if weight is not None:
        x = x * weight.double() / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt()
    n, f, out = case["rotated"], case["factor"], x.clone()
    base = case["base"] * (f ** (n / (n - 2.0)) if case["scaling"] == "ntk" else 1.0)
    gain = 1.0
    for i in range(n // 2):
        w = 1.0 / base ** (2.0 * i / n)
        if case["scaling"] == "linear":
            w /= f
        elif case["scaling"] == "yarn":
            gain = 1.0 + 0.1 * math.log(f)
            ends = [n / 2.0 * (math.log(4096.0) - math.log(2 * math.pi * t)) / math.log(base) for t in (32.0, 1.0)]
            lo, hi = max(0, math.floor(ends[0])), min(n - 1, math.ceil(ends[1]))
            share = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            w = share * w / f + (1.0 - share) * w
        a, b = (i, i + n // 2) if case["style"] == "half" else (2 * i, 2 * i + 1)
        z = torch.polar(torch.full_like(positions, gain, dtype=torch.float64), positions.double() * (-w if case.get("inverse") else w))
        y = torch.complex(x[..., a], x[..., b]) * z[:, None]
        out[..., a], out[..., b] = y.real, y.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _turned(case, s["x"], s["positions"], s["q_norm"])
    groups, shared, lens = _sizes(case)
    table, page, dev = s["table"].cpu().tolist(), case["page"], s["k"].device
    if case["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        pos = torch.cat([torch.arange(n - new, n, device=dev) for n, new in lens])
        keys, row = _turned(case, s["k_new"], pos, s["k_norm"]), 0
        for b, (n, new) in enumerate(lens):
            p = n - new
            while p < n:
                m = min(page - p % page, n - p)
                t = row + p - (n - new)
                k[0, table[b][p // page], :, p % page:p % page + m] = keys[t:t + m].transpose(0, 1)
                v[0, table[b][p // page], :, p % page:p % page + m] = s["v_new"][t:t + m].double().transpose(0, 1)
                p += m
            row += new
        return (k, v) if s["q"] is None else (k, v, _turned(case, s["q"], pos, s["q_norm"]))
    r, outs, row, g = case["q_heads"] // case["kv_heads"], [], 0, 0
    for b, (n, new) in enumerate(lens):
        g += b == groups[g + 1]
        first, j = groups[g], torch.arange(n, device=dev)
        at = torch.tensor([table[first if x < shared[g] else b][x // page] for x in range(n)], device=dev)
        hidden = j[None, :] > torch.arange(n - new, n, device=dev)[:, None]
        out = torch.zeros(new, case["q_heads"], case["dim"], dtype=torch.float64, device=dev)
        for i in range(case["kv_heads"]):
            kk, vv = (x[0, at, i, j % page].double() for x in (s["k"], s["v"]))
            heads = slice(i * r, (i + 1) * r)
            a = torch.einsum("thd,jd->htj", s["q"][row:row + new, heads].double(), kk) * case["dim"] ** -0.5
            a = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
            out[:, heads] = torch.einsum("htj,jd->thd", a, vv)
        outs.append(out)
        row += new
    return torch.cat(outs)
