"""The tensor-core kernel of prompts where it can go wrong: every call here is one that takes it, by
PagedKv.prompt_kernel, unless the test says otherwise."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
import kv_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ctx(bfv):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=0)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, *shape, dtype=BF):
    return torch.randn(*shape, generator=gen).to(dtype)


def check(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"error is {over:.3f} of the bound"


class Session:
    """lens: (length, new tokens) per sequence.  Values that no query sees are NaN in the cache."""

    def __init__(self, bfv, ctx, dtype, lens, heads, group, dim, page, window=0, sinks=0, layout="hnd", width=None, seed=7,
                 spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.ctx, self.lens, self.heads, self.group, self.dim = ctx, lens, heads, group, dim
        self.window, self.sinks, self.scale = window, sinks, dim ** -0.5
        self.cache = R.Cache(heads, dim, page, dtype, [n for n, _ in lens], 1, layout, width=width)
        self.held = []
        for s, (length, new) in enumerate(lens):
            k, v = randn(gen, length, heads, dim, dtype=dtype), randn(gen, length, heads, dim, dtype=dtype)
            self.held.append((k, v))
            old = min(new, length)
            seen = (R.visible(range(length - old, length), length, window, sinks).any(0) if old
                    else torch.zeros(length, dtype=torch.bool))
            self.cache.put(s, k, v, 0, only=seen)
            if window:
                self.cache.trim(s, length - new, window, sinks)
        self.kv = bfv.PagedKv(ctx, self.cache.k, self.cache.v)
        self.table, self.lengths = self.cache.table.cuda(), ints([n for n, _ in lens])
        self.starts = ints([0] + torch.tensor([n for _, n in lens]).cumsum(0).tolist())
        self.q = randn(gen, sum(n for _, n in lens), heads * group, dim, dtype=dtype) * spread
        self.q_dev = self.q.cuda()

    def call(self, kernel="tiles", q=None, starts=None, table=None, lengths=None):
        q = self.q_dev if q is None else q
        table = self.table if table is None else table
        assert self.kv.prompt_kernel(q, table, self.window, self.sinks) == kernel
        return self.kv.prompt(q, self.starts if starts is None else starts, table, self.lengths if lengths is None else lengths,
                              window=self.window, sinks=self.sinks)

    def rows(self, s):
        at = sum(n for _, n in self.lens[:s])
        return slice(at, at + self.lens[s][1])

    def check(self, got, seqs=None, q=None):
        q = self.q if q is None else q
        for s in range(len(self.lens)) if seqs is None else seqs:
            length, new = self.lens[s]
            mine, old = self.rows(s), min(new, length)
            out = got[mine]
            assert (out[:new - old] == 0).all()  # rows before the sequence's begin
            want, bound = R.attention(q[mine][new - old:], *self.held[s], length, self.window, self.sinks, self.scale,
                                      two_terms=False)
            check(out[new - old:], want, bound)

    def recorded(self, bfv):
        with pytest.raises(bfv.BfvGpuError, match="E_KV_TABLE"):
            self.ctx.check()
        assert self.ctx.check() == 0


MASKS = [
    # dtype, (length, new), kv_heads, group, dim, page, window, sinks, layout
    (BF, [(1500, 1500)], 1, 4, 96, 16, 1, 0, "hnd"),
    (FP, [(1100, 1100)], 1, 5, 128, 16, 1, 1, "hnd"),
    (FP, [(2500, 2100)], 2, 4, 64, 64, 2, 17, "nhd"),
    (BF, [(2000, 2000)], 1, 2, 128, 16, 64, 4, "hnd"),
    (BF, [(2500, 2300)], 1, 1, 128, 64, 130, 300, "hnd"),     # first tokens that reach into the window
    (FP, [(1800, 1700), (140, 100), (129, 128)], 2, 2, 64, 32, 127, 129, "gaps"),
    (BF, [(1500, 1200)], 1, 17, 64, 16, 50, 2, "hnd"),
    (BF, [(64, 0), (900, 900), (0, 0), (30, 2), (700, 300)], 2, 2, 128, 16, 0, 0, "hnd"),   # nothing new, nothing at all
    (FP, [(900, 900), (500, 0), (600, 600)], 2, 3, 72, 32, 256, 0, "nhd"),
    (FP, [(300, 300)], 2, 40, 8, 16, 0, 0, "hnd"),
    (BF, [(400, 400)], 1, 9, 104, 128, 128, 128, "nhd"),
]


@pytest.mark.parametrize("case", MASKS, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_masks(bfv, ctx, case):
    dtype, lens, heads, group, dim, page, window, sinks, layout = case
    s = Session(bfv, ctx, dtype, lens, heads, group, dim, page, window, sinks, layout)
    got = s.call()
    assert torch.equal(got, s.call())
    assert ctx.check() == 0
    s.check(got)


@pytest.mark.parametrize("group,new,length", [(127, 60, 300), (128, 70, 300), (129, 60, 300), (200, 40, 300), (300, 31, 200),
                                              (1024, 9, 130)])
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (FP, 64)])
def test_large_groups(bfv, ctx, group, new, length, dtype, dim):
    """Query heads of one token that fill a row tile or more than one: their queries are loaded row by row."""
    s = Session(bfv, ctx, dtype, [(length, new), (length - 1, new - 1)], 2, group, dim, 16)
    got = s.call()
    assert torch.equal(got, s.call())
    assert ctx.check() == 0
    s.check(got)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides_of_queries(bfv, ctx, dtype):
    """Tokens inside the heads: the kernel's loads follow them.  Broadcast over heads or tokens: the row kernel's do."""
    gen = torch.Generator().manual_seed(4)
    s = Session(bfv, ctx, dtype, [(900, 700), (800, 800)], 2, 2, 64, 16)
    turned = randn(gen, 4, 1500, 64, dtype=dtype).cuda().transpose(0, 1)
    s.check(s.call(q=turned), q=turned.cpu())
    one = randn(gen, 1500, 1, 64, dtype=dtype).cuda()
    for q in (one.expand(1500, 4, 64), one[:1].expand(1500, 4, 64)):
        s.check(s.call("rows", q=q), q=q.cpu())
    assert ctx.check() == 0


@pytest.mark.parametrize("new,heads,group,dim,width", [(3000, 4, 2, 64, None), (3060, 4, 2, 64, None), (1700, 2, 3, 128, None),
                                                       (600, 1, 2, 128, 300), (631, 1, 2, 64, 300)])
def test_more_queries_than_tokens(bfv, ctx, new, heads, group, dim, width):
    """Rows before the sequence's begin see nothing: zeros, in units without a key, in row tiles without one, and in row
    tiles of which some rows have one; with a wide table also where the launch has several parts."""
    s = Session(bfv, ctx, BF, [(30, new), (40, 40), (0, 50)], heads, group, dim, 16, width=width)
    got = s.call()
    assert torch.equal(got, s.call())
    assert ctx.check() == 0
    s.check(got)


def test_infinite_and_nan_keys(bfv, ctx):
    """A visible NaN reaches its own heads and sequence, nothing else; a visible -inf score weighs 0."""
    s = Session(bfv, ctx, FP, [(600, 500)] * 3, 2, 2, 128, 16)
    s.q = s.q.abs() + 0.5
    s.q_dev = s.q.cuda()
    good = s.call()
    p, r = s.cache.where(1)
    s.cache.v[0, p[50], 0, r[50], 3] = math.nan
    p, r = s.cache.where(2)
    s.cache.k[0, p[50], :, r[50], 3] = -math.inf
    got = s.call()
    assert ctx.check() == 0
    s.check(got, seqs=[0])
    assert torch.equal(got[s.rows(0)], good[s.rows(0)])
    nan = torch.isnan(got[s.rows(1)])
    assert nan[:, :2, 3].all() and nan.sum() == 500 * 2
    keep = torch.arange(600) != 50
    seen = R.visible(range(100, 600), 600, 0, 0)[:, keep]
    for h in range(4):
        k, v = s.held[2]
        want, bound = R.rows(s.q[s.rows(2), h], k[keep][:, h // 2], v[keep][:, h // 2], seen, s.scale, False)
        check(got[s.rows(2)][:, h], want, bound)


KINDS = [
    # units of few sequences by their keys; of many in the sequences' order; keys in parts
    dict(lens=[(900, 600), (900, 600)], width=None),
    dict(lens=[(900, 600), (900, 600)] + [(20, 9)] * 38, width=None),
    dict(lens=[(5000, 200), (5000, 200)], width=None),
]


@pytest.mark.parametrize("kind", KINDS, ids=["ranked", "many", "parts"])
def test_bad_tables_and_lengths_are_recorded_not_followed(bfv, ctx, kind):
    s = Session(bfv, ctx, BF, kind["lens"], 2, 2, 128, 16)
    good = s.call()
    assert ctx.check() == 0
    for bad in (-1, s.cache.k.shape[1], 2 ** 31 - 1, -2 ** 31):
        for slot in (1, 40):
            table = s.cache.table.clone()
            table[1, slot] = bad
            got = s.call(table=table.cuda())
            s.recorded(bfv)
            assert torch.equal(got[s.rows(0)], good[s.rows(0)])
    for bad in (-3, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        lengths = s.lengths.clone()
        lengths[1] = bad
        got = s.call(lengths=lengths)
        s.recorded(bfv)
        assert torch.equal(got[s.rows(0)], good[s.rows(0)])


@pytest.mark.parametrize("kind", KINDS, ids=["ranked", "many", "parts"])
def test_bad_starts_are_recorded_not_followed(bfv, ctx, kind):
    s = Session(bfv, ctx, BF, kind["lens"], 2, 2, 128, 16)
    tokens, a = s.q.shape[0], kind["lens"][0][1]
    for first, second, third in ((0, a, tokens + 1), (0, -5, tokens), (0, tokens + 100, tokens), (0, a, 2 ** 31 - 1),
                                 (-2 ** 31, a, tokens), (a, 0, tokens), (0, a, -2 ** 31), (0, 0, 0), (1, a, tokens),
                                 (0, a, a)):
        starts = s.starts.clone()
        starts[0], starts[1], starts[2] = first, second, third
        if len(kind["lens"]) > 2:
            starts[3:] = third
        s.call(starts=starts)
        s.recorded(bfv)
    good = s.call()
    assert ctx.check() == 0
    s.check(good)


def test_graph_of_prompts(bfv, ctx):
    """Captured once, replayed with other queries, lengths, starts and tables."""
    a = Session(bfv, ctx, BF, [(900, 600), (700, 600)], 2, 2, 128, 16)
    tables = torch.stack([a.table, a.table.flip(0)])
    starts, lengths, table, q = a.starts.clone(), a.lengths.clone(), a.table.clone(), a.q_dev.clone()
    assert a.kv.prompt_kernel(q, table) == "tiles"
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.kv.prompt(q, starts, table, lengths, out=out)
    for i, (cut, n) in enumerate([(600, (900, 700)), (300, (700, 900)), (1200, (900, 5)), (0, (3, 900))]):
        starts.copy_(ints([0, cut, 1200]))
        lengths.copy_(ints(n))
        table.copy_(tables[i % 2])
        q.copy_(a.q_dev * (1 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = a.kv.prompt(q, starts, table, lengths)
        assert ctx.check() == 0
        assert torch.equal(got, want)
        for s, (lo, hi) in enumerate(((0, cut), (cut, 1200))):
            k, v = a.held[s if i % 2 == 0 else 1 - s]
            new, length = hi - lo, n[s]
            k, v = k[:length], v[:length]
            old = min(new, length)
            assert (got[lo:hi - old] == 0).all()
            o, b = R.attention(q[hi - old:hi].cpu(), k, v, length, 0, 0, a.scale, two_terms=False)
            check(got[hi - old:hi], o, b)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_large_scores(bfv, ctx, dtype):
    """Scores to about +-200 over many key tiles: the reference exponent has to follow them."""
    s = Session(bfv, ctx, dtype, [(1500, 900), (700, 700)], 2, 3, 64, 32, spread=40.0)
    got = s.call()
    assert torch.equal(got, s.call())
    assert ctx.check() == 0
    s.check(got)
