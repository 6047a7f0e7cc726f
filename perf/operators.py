"""The operators of the paged key-value cache, as they are timed: one pass each of

* ``decode``  attention of one new token per sequence over the cache's pages;
* ``prompt``  attention of a prompt (or of its next chunk) over the pages, causal, optionally with a sliding
              window and first tokens that stay visible;
* ``append``  new keys and values written into the pages of their sequences;
* ``fork``    sequences that continue another one: shared full pages, a copy of the partly filled last page;
* ``move``    pages copied to the holes of the cache (compaction), and the tables that name them.

Shapes: K and V [layers][pages][kv_heads][page][dim], table [sequences][width] page numbers (-1: no page),
lengths [sequences].  ``own`` False: elementary torch operations in 32 bits.  ``own`` True: the calls of
``bfvgpu.PagedKv``.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _case(name, op, **kw):
    c = dict(op=op, seqs=1, length=512, ragged=False, new=1, q_heads=16, kv_heads=8, dim=128, page=16, dtype="bf16",
             source="bf16", layout="hnd", window=0, sinks=0, layers=1, moved=0)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the first token of a decode after a 512-token prefill: 16 query heads, 8 key heads of 128 (the layer whose
        # q/k/v call is 1024 -> 4096); latency
        _case("decode first token", "decode", length=513),
        # a serving batch at mixed lengths
        _case("decode batch", "decode", seqs=64, length=4096, ragged=True),
        # one long document, few key heads: the length has to be split
        _case("decode long", "decode", length=131071, q_heads=32, kv_heads=4, page=64, dtype="fp16"),
        # many sessions with a window and four first tokens; pages outside the window are gone
        _case("decode window", "decode", seqs=96, length=16384, ragged=True, q_heads=16, kv_heads=2, dim=64, page=32,
              window=1024, sinks=4),
        # the last 16-token tile of a 512-token prefill, the tile of the linear layers' calls; latency
        _case("prompt tile", "prompt", length=512, new=16),
        # eight 512-token prefills
        _case("prompt batch", "prompt", seqs=8, length=512, new=512),
        # the next chunks of mixed sessions: odd lengths, three query heads per key head, pages with the heads inside
        _case("prompt chunks", "prompt", seqs=6, length=8192, new=1024, ragged=True, q_heads=12, kv_heads=4, dim=64,
              page=32, dtype="fp16", layout="nhd"),
        # a long document with a window and four first tokens
        _case("prompt window", "prompt", length=8191, new=8191, page=64, window=1024, sinks=4),
        # the keys and values of one decode step of 64 sequences, one layer
        _case("append step", "append", seqs=64, length=4096, ragged=True),
        # those of prompts, computed in 32 bits and stored in 16
        _case("append prompt", "append", seqs=8, length=4096, new=4096, ragged=True, source="f32"),
        # one retrieved document, sixteen answers: 28 layers
        _case("fork answers", "fork", seqs=17, length=1000, layers=28, moved=16),
        # compaction of the same cache after half of its sequences ended
        _case("move pages", "move", seqs=16, length=512, ragged=True, layers=28, moved=256),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    largest = {}
    for c in listed():
        w, g = work(c), _padded(c)
        m = largest.setdefault(c["op"], [0, 0, 0])
        largest[c["op"]] = [max(m[0], w["bytes"]), max(m[1], w["flops"]), max(m[2], g)]
    while True:
        op = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "prompt", "append", "fork", "move"])
        kv = rng.choice([1, 2, 3, 4, 8])
        c = _case(None, op, kv_heads=kv, q_heads=kv * rng.choice([1, 2, 3, 4, 5, 8]), dim=rng.choice([64, 72, 96, 128, 128]),
                  page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "fp16"]), layout=rng.choice(["hnd", "nhd"]),
                  ragged=rng.random() < 0.7)
        c["source"] = rng.choice([c["dtype"], "f32"])
        if op == "decode":
            c.update(seqs=_log(rng, 1, 128), length=_log(rng, 1, 131071))
        elif op == "prompt":
            c.update(seqs=_log(rng, 1, 16), length=_log(rng, 1, 8192))
            c["new"] = c["length"] if rng.random() < 0.4 else _log(rng, 1, c["length"])
        elif op == "append":
            c.update(seqs=_log(rng, 1, 128), length=_log(rng, 1, 8192))
            c["new"] = 1 if rng.random() < 0.4 else _log(rng, 1, c["length"])
        else:
            c.update(layers=_log(rng, 1, 28), length=_log(rng, 2, 1024), seqs=_log(rng, 2, 32))
            c["moved"] = rng.randint(1, c["seqs"] - 1) if op == "fork" else _log(rng, 1, 256)
        if op in ("decode", "prompt") and rng.random() < 0.4:
            c.update(window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 17]))
        w, (b, f, g) = work(c), largest[op]
        if w["bytes"] <= b and w["flops"] <= f and _padded(c) <= g:
            return c


def _lengths(case):
    """(length, new tokens) of each sequence: the sizes of a case, the same for every seed."""
    rng = random.Random("%(op)s %(seqs)d %(length)d %(new)d" % case)
    out = []
    for s in range(case["seqs"]):
        if not case["ragged"] or s == 0:
            out.append((case["length"], case["new"]))
        elif case["op"] in ("prompt", "append") and case["new"] == case["length"]:
            n = rng.randint(1, case["length"])
            out.append((n, n))
        else:
            n = rng.randint(1, case["length"])
            out.append((n, min(n, rng.randint(1, case["new"]))))
    return out


def _padded(case):
    """Size of the padded arrays of the plain form."""
    kv = case["seqs"] * case["length"] * case["kv_heads"] * case["dim"]
    if case["op"] == "prompt":
        return max(kv, case["seqs"] * case["new"] * case["length"] * case["q_heads"])
    return kv if case["op"] == "decode" else 0 if case["op"] == "append" else _pages(case)[1] * _page_bytes(case)


def _visible(p, window, sinks):
    """Number of keys that a query at position p sees."""
    if not window or window > p:
        return p + 1
    return window + min(sinks, p + 1 - window)


def _pages(case):
    """(pages in use, pages in the cache)."""
    used = sum(-(-n // case["page"]) for n, _ in _lengths(case))
    if case["op"] == "fork":
        return used, used + case["moved"] + 3
    if case["op"] == "move":
        return used + case["moved"], used + 2 * case["moved"] + 3
    return used, used + 3


def _page_bytes(case):
    return case["kv_heads"] * case["page"] * case["dim"] * 2


def work(case):
    h, g, d = case["q_heads"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    if case["op"] in ("fork", "move"):
        n = case["moved"]
        if case["op"] == "fork" and case["length"] % case["page"] == 0:
            n = 0
        rows = case["seqs"] * -(-case["length"] // case["page"]) * 4
        return {"bytes": 2 * 2 * case["layers"] * n * _page_bytes(case) + 2 * rows, "flops": 0}
    if case["op"] == "append":
        tokens = sum(n for _, n in lens)
        return {"bytes": 2 * tokens * g * d * (2 + (4 if case["source"] == "f32" else 2)), "flops": 0}
    w, s = case["window"], case["sinks"]
    pairs = keys = 0
    for length, new in lens:
        new = new if case["op"] == "prompt" else 1
        first = length - new
        # positions below the window see all before them; from there on the count is constant
        full = min(length, max(first, w)) if w else length
        pairs += (full * (full + 1) - first * (first + 1)) // 2 if full > first else 0
        at = max(full, first)
        if w and at < length:
            top = max(at, min(length, w + s))
            pairs += sum(_visible(p, w, s) for p in range(at, top)) + (length - top) * (w + s)
        keys += length if not w or first < w else (length - first - 1) + _visible(first, w, s)
    tokens = sum(n for _, n in lens) if case["op"] == "prompt" else len(lens)
    return {"bytes": 2 * 2 * keys * g * d + 2 * 2 * tokens * h * d, "flops": 4 * pairs * h * d}


# ----------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt, src = DTYPES[case["dtype"]], DTYPES[case["source"]]
    h, g, d, page, layers = case["q_heads"], case["kv_heads"], case["dim"], case["page"], case["layers"]
    lens = _lengths(case)
    _, total = _pages(case)
    rand = lambda *s: torch.randn(*s, device=dev, generator=gen, dtype=torch.float32 if case["op"] == "append" else dt)  # noqa: E731
    shape = (layers, total, g, page, d) if case["layout"] == "hnd" else (layers, total, page, g, d)
    k, v = rand(*shape).to(dt), rand(*shape).to(dt)
    if case["layout"] == "nhd":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    # pages in the order of a cache that has been in use: any page may hold any part
    perm = torch.randperm(total, device=dev, generator=gen).to(torch.int32)
    width = -(-max(n for n, _ in lens) // page) + 1
    seqs = len(lens)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device=dev)
    lengths = torch.tensor([n for n, _ in lens], dtype=torch.int32, device=dev)
    counts = (lengths + (page - 1)) // page
    at = torch.arange(width, device=dev, dtype=torch.int32)
    held = at < counts[:, None]
    used = int(sum(-(-n // page) for n, _ in lens))
    table[held] = perm[:used]
    state = dict(op=case["op"], k=k, v=v, table=table, lengths=lengths, window=case["window"], sinks=case["sinks"],
                 page=page, scale=1.0 / math.sqrt(d))
    if case["op"] in ("decode", "prompt"):
        if case["window"]:  # the pages that no query of this pass sees are gone
            first = lengths - torch.tensor([n if case["op"] == "prompt" else 1 for _, n in lens], device=dev, dtype=torch.int32)
            gone = ((at + 1) * page <= (first - case["window"] + 1)[:, None]) & (at * page >= case["sinks"])
            table[gone] = -1
        tokens = sum(n for _, n in lens) if case["op"] == "prompt" else seqs
        # the queries lie in the rows of a joint q/k/v product, as the layer's call leaves them
        state["q"] = rand(tokens, (h + 2 * g) * d)[:, :h * d].unflatten(1, (h, d))
    if case["op"] in ("prompt", "append"):
        new = torch.tensor([n for _, n in lens], device=dev)
        state["starts"] = torch.cat([new.new_zeros(1), new.cumsum(0)]).to(torch.int32)
        state["most"] = max(n for _, n in lens)
    if case["op"] == "append":
        row = rand(sum(n for _, n in lens), (h + 2 * g) * d).to(src)
        state["k_new"] = row[:, h * d:(h + g) * d].unflatten(1, (g, d))
        state["v_new"] = row[:, (h + g) * d:].unflatten(1, (g, d))
    if case["op"] == "fork":  # children: the last rows; they continue the first sequence
        n = case["moved"]
        state["parents"] = torch.zeros(n, dtype=torch.int32, device=dev)
        state["children"] = torch.arange(seqs - n, seqs, dtype=torch.int32, device=dev)
        state["fresh"] = perm[used:used + n].contiguous()
    if case["op"] == "move":  # pages in use, in rising order, and the holes that take them
        n = case["moved"]
        pages = perm[:used]
        src_pages = pages[torch.randperm(used, device=dev, generator=gen)[:min(n, used)]]
        more = perm[used:used + n - src_pages.numel()]
        state["src"] = torch.cat([src_pages, more]).sort().values.contiguous()
        state["dst"] = perm[used + n:used + 2 * n].contiguous()
    return state


# ------------------------------------------------------------------------------------------- plain forms
def _sequence_of(starts, tokens):
    t = torch.arange(tokens, device=starts.device)
    seq = torch.searchsorted(starts[1:].long(), t, right=True)
    return seq, t - starts.long()[seq]


def _keys_and_values(s):
    """K, V of every sequence [seqs][kv_heads][width * page][dim] in 32 bits."""
    table = s["table"].clamp(min=0).long()
    k, v = (x[0][table].transpose(1, 2).flatten(2, 3).float() for x in (s["k"], s["v"]))
    return k, v


def _attend(q, k, v, seen, scale):
    """q [B][G][rows][D], k, v [B][G][T][D], seen [B][1][rows][T]: softmax over the seen keys, 0 where there are none."""
    x = (q @ k.transpose(2, 3)) * scale
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total > 0, total, 1.0)


def _seen(pos, at, window, sinks):
    seen = at <= pos
    if window:
        seen = seen & ((at > pos - window) | (at < sinks))
    return seen


def _plain(s):
    op, table, lengths, page = s["op"], s["table"], s["lengths"], s["page"]
    if op in ("decode", "prompt"):
        k, v = _keys_and_values(s)
        q = s["q"].float()
        tokens, h, d = q.shape
        b, g = k.shape[:2]
        r = h // g
        at = torch.arange(k.shape[2], device=k.device)
    if op == "decode":
        pos = lengths.long()[:, None, None, None] - 1
        o = _attend(q.reshape(b, g, r, d), k, v, _seen(pos, at, s["window"], s["sinks"]), s["scale"])
        return o.reshape(b, h, d).to(s["q"].dtype)
    if op == "prompt":
        seq, i = _sequence_of(s["starts"], tokens)
        rows = q.new_zeros(b, s["most"], h, d)
        rows[seq, i] = q
        rows = rows.view(b, s["most"], g, r, d).permute(0, 2, 3, 1, 4).reshape(b, g, r * s["most"], d)
        new = (s["starts"][1:] - s["starts"][:-1]).long()
        pos = (lengths.long() - new)[:, None] + torch.arange(s["most"], device=q.device)
        seen = _seen(pos[:, None, :, None], at, s["window"], s["sinks"]).repeat(1, 1, r, 1)
        o = _attend(rows, k, v, seen, s["scale"])
        o = o.view(b, g, r, s["most"], d).permute(0, 3, 1, 2, 4)
        return o[seq, i].reshape(tokens, h, d).to(s["q"].dtype)
    if op == "append":
        k, v = s["k"][0], s["v"][0]
        seq, i = _sequence_of(s["starts"], s["k_new"].shape[0])
        new = (s["starts"][1:] - s["starts"][:-1]).long()
        pos = (lengths.long() - new)[seq] + i
        at = table[seq, pos // page].long()
        k[at, :, pos % page] = s["k_new"].to(k.dtype)
        v[at, :, pos % page] = s["v_new"].to(v.dtype)
        return s["k"], s["v"]
    if op == "fork":
        parents, children, fresh = (s[x].long() for x in ("parents", "children", "fresh"))
        length = lengths[parents]
        rows = table[parents]
        last = (length // page).long().clamp(max=table.shape[1] - 1)[:, None]
        tail = rows.gather(1, last)[:, 0].long()
        part = length % page > 0
        to = torch.where(part, fresh, tail)
        table[children] = rows.scatter(1, last, to[:, None].int())
        lengths[children] = length
        # a full last page is shared: its "copy" is onto any page's own place
        safe = torch.where(part, tail, 0)
        to = torch.where(part, to, 0)
        s["k"][:, to] = s["k"][:, safe]
        s["v"][:, to] = s["v"][:, safe]
        return s["k"], s["v"], table, lengths
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    to = torch.arange(s["k"].shape[1], device=table.device, dtype=torch.int32)
    to[src] = s["dst"]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    return s["k"], s["v"], table


# --------------------------------------------------------------------------------- the framework's calls
_kept = {}


def _cache(s):
    """The cache object and the context that a program holds for as long as it holds its pages."""
    if "cache" not in s:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "privacy-rag_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import bfvgpu
        if "ctx" not in _kept:  # the small transform context: n = 4096, 36/36/37-bit primes
            _kept["ctx"] = bfvgpu.Context(4096, bfvgpu.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=0)
        s["cache"] = bfvgpu.PagedKv(_kept["ctx"], s["k"], s["v"])
    return s["cache"]


def run(state):
    if not own:
        return _plain(state)
    s, c = state, _cache(state)
    op = s["op"]
    if op == "decode":
        return c.decode(s["q"], s["table"], s["lengths"], window=s["window"], sinks=s["sinks"], scale=s["scale"])
    if op == "prompt":
        return c.prompt(s["q"], s["starts"], s["table"], s["lengths"], window=s["window"], sinks=s["sinks"], scale=s["scale"])
    if op == "append":
        c.append(s["k_new"], s["v_new"], s["starts"], s["table"], s["lengths"])
        return s["k"], s["v"]
    if op == "fork":
        c.fork(s["parents"], s["children"], s["fresh"], s["table"], s["lengths"])
        return s["k"], s["v"], s["table"], s["lengths"]
    c.move(s["src"], s["dst"], s["table"])
    return s["k"], s["v"], s["table"]


# --------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    lens, page = _lengths(case), case["page"]
    table = s["table"].cpu().tolist()
    if case["op"] in ("decode", "prompt"):
        r, outs, row = case["q_heads"] // case["kv_heads"], [], 0
        for b, (length, new) in enumerate(lens):
            new = new if case["op"] == "prompt" else 1
            out = torch.zeros(new, case["q_heads"], case["dim"], dtype=torch.float64, device="cuda")
            first = length - new
            lo = max(0, first - case["window"] + 1) if case["window"] else 0
            keys = sorted(set(range(lo, length)) | set(range(min(length, case["sinks"] if case["window"] else 0))))
            j = torch.tensor(keys, device="cuda")
            at = torch.tensor([table[b][x // page] for x in keys], device="cuda")
            p = torch.arange(first, length, device="cuda")
            off = j[None, :] > p[:, None]
            if case["window"]:
                off |= (j[None, :] <= p[:, None] - case["window"]) & (j[None, :] >= case["sinks"])
            for g in range(case["kv_heads"]):
                kk = s["k"][0, at, g, j % page].double()
                vv = s["v"][0, at, g, j % page].double()
                for i in range(g * r, (g + 1) * r):
                    a = s["q"][row:row + new, i].double().mm(kk.t()).mul_(case["dim"] ** -0.5)
                    a[off] = -math.inf
                    out[:, i] = torch.softmax(a, 1).mm(vv)
            outs.append(out)
            row += new
        return torch.cat(outs)
    k, v = s["k"].double(), s["v"].double()
    if case["op"] == "append":
        row = 0
        for b, (length, new) in enumerate(lens):
            for p in range(length - new, length, 1):
                if p % page == 0 or p == length - new:
                    n = min(page - p % page, length - p)
                    t = row + p - (length - new)
                    for x, y in ((k, s["k_new"]), (v, s["v_new"])):
                        x[0, table[b][p // page], :, p % page:p % page + n] = y[t:t + n].double().transpose(0, 1)
            row += new
        return k, v
    lengths = list(n for n, _ in lens)
    if case["op"] == "fork":
        for p, c, f in zip(*(s[x].cpu().tolist() for x in ("parents", "children", "fresh"))):
            table[c], lengths[c] = list(table[p]), lengths[p]
            if lengths[p] % page:
                at = lengths[p] // page
                table[c][at] = f
                k[:, f], v[:, f] = k[:, table[p][at]], v[:, table[p][at]]
        return k, v, torch.tensor(table, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)
    to = dict(zip(s["src"].cpu().tolist(), s["dst"].cpu().tolist()))
    for a, b in to.items():
        k[:, b], v[:, b] = k[:, a], v[:, a]
    return k, v, torch.tensor([[to.get(x, x) for x in row] for row in table], dtype=torch.int32)
