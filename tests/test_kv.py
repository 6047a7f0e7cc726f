"""Paged key-value cache without a GPU: the refusals of the C ABI (on a host-only context: every
argument is checked before the device), the scratch sizes, and the book-keeping of the pages."""
from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import pytest

ARGUMENT, SHAPE, DEVICE = 1, 3, 10


@pytest.fixture(scope="module")
def host(bfv):
    return bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=-1)


def desc(bfv, **over):
    from bfvgpu._lib import KvDesc
    page, heads, dim, pages = 16, 2, 64, 8
    d = dict(k=0x10000, v=0x20000, dtype=0, layers=2, pages=pages, heads=heads, page_tokens=page, dim=dim,
             layer_stride=pages * heads * page * dim, page_stride=heads * page * dim, head_stride=page * dim,
             token_stride=dim)
    d.update(over)
    return KvDesc(*[d[f] for f, _ in KvDesc._fields_])


P = 0x30000  # a well-aligned address that nothing reads


def calls(bfv, host, cache, **over):
    """Every entry point with arguments that are right but for `over`: {name: (status, message)}."""
    a = dict(layer=0, p=P, src=0, ts=128, hs=64, tokens=4, starts=P, table=P, width=3, lengths=P, seqs=2, heads=4,
             window=0, sinks=0, scale=0.125, scratch=P, out=P, rows=4, count=2, k=P)
    a.update(over)
    L, h = bfv.lib(), host.handle if over.get("ctx", 1) else None
    ref = ctypes.byref(cache) if cache is not None else None
    got = {}

    def note(name, rc):
        got[name] = (rc, L.bfvgpu_last_error().decode())

    note("append", L.bfvgpu_kv_append_device(h, ref, a["layer"], a["k"], a["p"], a["src"], a["ts"], a["hs"], a["tokens"],
                                             a["starts"], a["table"], a["width"], a["lengths"], a["seqs"], None))
    note("decode", L.bfvgpu_kv_decode_device(h, ref, a["layer"], a["p"], a["ts"], a["hs"], a["heads"], a["table"],
                                             a["width"], a["lengths"], a["seqs"], a["window"], a["sinks"], a["scale"],
                                             a["scratch"], a["out"], None))
    note("prompt", L.bfvgpu_kv_prompt_device(h, ref, a["layer"], a["p"], a["ts"], a["hs"], a["heads"], a["tokens"],
                                             a["starts"], a["table"], a["width"], a["lengths"], a["seqs"], a["window"],
                                             a["sinks"], a["scale"], a["scratch"], a["out"], None))
    note("fork", L.bfvgpu_kv_fork_device(h, ref, a["p"], a["p"], a["p"], a["count"], a["table"], a["rows"], a["width"],
                                         a["lengths"], None))
    note("move", L.bfvgpu_kv_move_device(h, ref, a["p"], a["p"], a["count"], a["table"], a["rows"], a["width"], None))
    return got


def test_right_arguments_reach_the_device_check(bfv, host):
    for cache in (desc(bfv), desc(bfv, dtype=1), desc(bfv, head_stride=64, token_stride=128),
                  desc(bfv, dim=8, token_stride=64), desc(bfv, page_tokens=256, page_stride=1 << 20, head_stride=1 << 15),
                  desc(bfv, pages=2, layers=1, layer_stride=0, heads=1, head_stride=0)):
        for name, (rc, text) in calls(bfv, host, cache, src=cache.dtype).items():
            assert (rc, text) == (DEVICE, "E_BFVGPU_HOST_ONLY_CONTEXT"), name


@pytest.mark.parametrize("over,code,text", [
    (dict(k=0), ARGUMENT, "E_KV_ARGUMENT"), (dict(v=0), ARGUMENT, "E_KV_ARGUMENT"),
    (dict(dtype=2), ARGUMENT, "E_KV_DTYPE"), (dict(dtype=-1), ARGUMENT, "E_KV_DTYPE"),
    (dict(layers=0), SHAPE, "E_KV_SHAPE"), (dict(pages=0), SHAPE, "E_KV_SHAPE"), (dict(heads=0), SHAPE, "E_KV_SHAPE"),
    (dict(heads=1025), SHAPE, "E_KV_SHAPE"),
    (dict(dim=0), SHAPE, "E_KV_DIM"), (dict(dim=60), SHAPE, "E_KV_DIM"), (dict(dim=136), SHAPE, "E_KV_DIM"),
    (dict(page_tokens=8), SHAPE, "E_KV_PAGE_TOKENS"), (dict(page_tokens=48), SHAPE, "E_KV_PAGE_TOKENS"),
    (dict(page_tokens=512), SHAPE, "E_KV_PAGE_TOKENS"),
    (dict(token_stride=0), SHAPE, "E_KV_STRIDE"), (dict(page_stride=-2048), SHAPE, "E_KV_STRIDE"),
    (dict(layer_stride=1 << 40), SHAPE, "E_KV_STRIDE"),
    (dict(token_stride=68), ARGUMENT, "E_KV_ALIGNMENT"), (dict(head_stride=1025), ARGUMENT, "E_KV_ALIGNMENT"),
    (dict(k=0x10008), ARGUMENT, "E_KV_ALIGNMENT"), (dict(v=0x20002), ARGUMENT, "E_KV_ALIGNMENT"),
])
def test_cache_descriptions_refused(bfv, host, over, code, text):
    for name, got in calls(bfv, host, desc(bfv, **over)).items():
        assert got == (code, text), name


def test_null_cache_and_context(bfv, host):
    for name, got in calls(bfv, host, None).items():
        assert got == (ARGUMENT, "E_KV_ARGUMENT"), name
    for name, got in calls(bfv, host, desc(bfv), ctx=0).items():
        assert got == (ARGUMENT, "E_BFVGPU_ARGUMENT"), name


@pytest.mark.parametrize("over,names,code,text", [
    (dict(layer=-1), "append decode prompt", SHAPE, "E_KV_LAYER"),
    (dict(layer=2), "append decode prompt", SHAPE, "E_KV_LAYER"),
    (dict(heads=3), "decode prompt", SHAPE, "E_KV_HEADS"),
    (dict(heads=0), "decode prompt", SHAPE, "E_KV_HEADS"),
    (dict(window=-1), "decode prompt", ARGUMENT, "E_KV_WINDOW"),
    (dict(sinks=-1), "decode prompt", ARGUMENT, "E_KV_WINDOW"),
    (dict(scale=0.0), "decode prompt", ARGUMENT, "E_KV_SCALE"),
    (dict(scale=-1.0), "decode prompt", ARGUMENT, "E_KV_SCALE"),
    (dict(scale=math.nan), "decode prompt", ARGUMENT, "E_KV_SCALE"),
    (dict(scale=math.inf), "decode prompt", ARGUMENT, "E_KV_SCALE"),
    (dict(width=1 << 27), "decode prompt", SHAPE, "E_KV_WIDTH"),
    (dict(tokens=1 << 32), "append prompt", SHAPE, "E_KV_SHAPE"),
    (dict(seqs=1 << 31), "append decode prompt", SHAPE, "E_KV_SHAPE"),
    (dict(starts=None), "append", SHAPE, "E_KV_STARTS"),
    (dict(starts=None), "prompt", ARGUMENT, "E_KV_ARGUMENT"),
    (dict(src=1), "append", ARGUMENT, "E_KV_SOURCE_DTYPE"),
    (dict(src=3), "append", ARGUMENT, "E_KV_SOURCE_DTYPE"),
    (dict(count=5), "fork", SHAPE, "E_KV_SHAPE"),
    (dict(count=9), "move", SHAPE, "E_KV_SHAPE"),
])
def test_calls_refused(bfv, host, over, names, code, text):
    got = calls(bfv, host, desc(bfv), **over)
    for name in names.split():
        assert got[name] == (code, text), name


def test_scratch_sizes(bfv, host):
    L, d = bfv.lib(), desc(bfv)
    ask = lambda seqs, width, window=0, heads=4: L.bfvgpu_kv_decode_scratch_words(  # noqa: E731
        host.handle, ctypes.byref(d), heads, seqs, width, window, 0)
    assert ask(2, 3) == 0 and ask(512, 1000) == 0     # short, or many sequences: no second join
    assert ask(1, 10000) > 0 and ask(1, 10000, window=100) == 0
    assert ask(1, 10000, heads=3) == 0                # refused arguments need none
    assert L.bfvgpu_kv_prompt_scratch_words(host.handle, ctypes.byref(d), 4, 3, 1, 3, 0, 0) == 0


# ---- book-keeping -----------------------------------------------------------------------------------
def consistent(book):
    held = book.table[book.table >= 0]
    refs = np.bincount(held, minlength=len(book.refs))
    assert np.array_equal(refs, book.refs)
    assert sorted(book._free) == np.flatnonzero(refs == 0).tolist()
    assert (book.table[~book.active] == -1).all() and (book.lengths[~book.active] == 0).all()
    for row in np.flatnonzero(book.active):
        n, p = int(book.lengths[row]), book.page_tokens
        assert (book.table[row, -(-n // p):] == -1).all()
        if n % p:  # tokens are only written to a page of one sequence
            assert book.refs[book.table[row, n // p]] == 1


def test_book_against_a_model(bfv):
    """Random sessions: every token keeps its own place, shared only where sequences share it."""
    rng = random.Random(5)
    for _ in range(20):
        page, pages, rows, width = rng.choice([4, 16]), 40, 6, 12
        book = bfv.PageBook(pages, page, rows, width)
        memory, told = {}, {}  # (page, offset) -> token id; row -> token ids (None: trimmed)
        for _ in range(120):
            act = rng.choice(["open", "extend", "extend", "extend", "fork", "free", "trim", "compact"])
            live = list(told)
            try:
                if act == "open":
                    told[book.open()] = []
                elif act == "extend" and live:
                    counts = {r: rng.randint(0, 9) for r in rng.sample(live, rng.randint(1, len(live)))}
                    before = {r: len(told[r]) for r in counts}
                    book.extend(counts)
                    for r, n in counts.items():
                        for j in range(before[r], before[r] + n):
                            told[r].append(rng.random())
                            memory[int(book.table[r, j // page]), j % page] = told[r][-1]
                elif act == "fork" and live:
                    r = rng.choice(live)
                    kids, fresh = book.fork(r, rng.randint(0, 2))
                    n = len(told[r])
                    for c, f in zip(kids, fresh):
                        told[c] = list(told[r])
                        assert (f >= 0) == (n % page != 0)
                        if f >= 0:
                            tail = int(book.table[r, n // page])
                            for o in range(n % page):
                                memory[f, o] = memory[tail, o]
                elif act == "free" and live:
                    r = rng.choice(live)
                    book.free(r)
                    del told[r]
                elif act == "trim" and live:
                    w, s = rng.randint(1, 30), rng.randint(0, 5)
                    book.trim(w, s)
                    for r in live:
                        for j in range(len(told[r])):
                            if book.table[r, j // page] < 0 and told[r][j] is not None:
                                assert j <= len(told[r]) - w and j >= s
                                told[r][j] = None
                elif act == "compact":
                    src, dst = book.compact()
                    assert src == sorted(src) and dst == sorted(dst) and not set(src) & set(dst)
                    for a, b in zip(src, dst):
                        for o in range(page):
                            if (a, o) in memory:
                                memory[b, o] = memory[a, o]
                    used = int((book.refs > 0).sum())
                    assert (book.refs[:used] > 0).all()
            except bfv.BfvGpuError as e:
                assert e.code == 14
            except ValueError as e:
                assert "E_KV_LENGTH" in str(e)
            consistent(book)
            for r, ids in told.items():
                assert book.lengths[r] == len(ids)
                for j, x in enumerate(ids):
                    if x is not None:
                        assert memory[int(book.table[r, j // page]), j % page] == x


def test_book_refusals_change_nothing(bfv):
    book = bfv.PageBook(4, 16, 3, 3)
    a = book.open()
    book.extend({a: 40})
    state = lambda: (book.table.copy(), book.lengths.copy(), book.refs.copy(), list(book._free), book.active.copy())  # noqa: E731
    before = state()

    def same():
        assert all(np.array_equal(x, y) for x, y in zip(before, state()))

    with pytest.raises(ValueError, match="E_KV_LENGTH"):
        book.extend({a: 9})
    same()
    with pytest.raises(ValueError, match="E_KV_LENGTH"):
        book.extend({a: -1})
    same()
    with pytest.raises(ValueError, match="E_KV_ROW"):
        book.extend({a: 1, 2: 1})
    same()
    with pytest.raises(ValueError, match="E_KV_ROW"):
        book.free(7)
    same()
    with pytest.raises(bfv.BfvGpuError, match="E_KV_PAGES"):
        book.fork(a, 2)
    same()
    with pytest.raises(bfv.BfvGpuError, match="E_KV_ROWS"):
        book.fork(a, 3)
    same()
    with pytest.raises(ValueError, match="E_KV_WINDOW"):
        book.trim(0, 1)
    same()
    for bad in ((0, 16, 1, 1), (1, 0, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0)):
        with pytest.raises(ValueError, match="E_KV_SHAPE"):
            bfv.PageBook(*bad)


def test_paged_kv_refuses_host_tensors(bfv, host):
    torch = pytest.importorskip("torch")
    z = torch.zeros(2, 3, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="E_KV_DEVICE"):
        bfv.PagedKv(host, z, z.clone())
    for k, v, text in ((z.float(), z.float(), "DTYPE"), (z, z[:1], "SHAPE"), (z, z.half(), "SHAPE"),
                       (z[..., ::2], z[..., ::2], "SHAPE"), (z, z.transpose(2, 3).contiguous().transpose(2, 3), "SHAPE"),
                       (z[0, 0], z[0, 0], "SHAPE")):
        with pytest.raises(ValueError, match="E_KV_" + text):
            bfv.PagedKv(host, k, v)


def test_calls_refuse_host_tensors(bfv):
    """The module of PagedKv's calls, on a made-up cache: what lies in host memory is refused before any use."""
    torch = pytest.importorskip("torch")
    import ctypes

    from bfvgpu import kvcache
    from bfvgpu._lib import KvDesc
    calls = kvcache._calls()
    desc = KvDesc(0x10000, 0x20000, 0, 1, 4, 2, 16, 64, 0, 2048, 1024, 64)
    cache = calls.open(ctypes.addressof(desc), 0)
    rows, ints = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(3, 2, dtype=torch.int32)
    for call in (lambda: calls.append(cache, None, rows, rows, None, table, ints, 0, None),
                 lambda: calls.fork(cache, None, ints, ints, ints, table, ints, None),
                 lambda: calls.move(cache, None, ints, ints, table, None),
                 lambda: calls.decode(cache, None, rows, table, ints, 0, 0, 0, None, None, None),
                 lambda: calls.prompt(cache, None, rows, ints, table, ints, 0, 0, 0, None, None, None)):
        with pytest.raises(ValueError, match="E_KV_SHAPE.*on the cache's device"):
            call()
    with pytest.raises(TypeError, match="a tensor is wanted"):
        calls.decode(cache, None, [1.0], table, ints, 0, 0, 0, None, None, None)
    with pytest.raises(TypeError, match="arguments"):
        calls.decode(cache, None, rows)
    with pytest.raises(ValueError):  # not a cache
        calls.move(object(), None, ints, ints, table, None)
    with pytest.raises(ValueError, match="E_KV_ARGUMENT"):
        calls.open(0, 0)
