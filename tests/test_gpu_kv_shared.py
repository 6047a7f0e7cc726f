"""Attention over tokens that groups of sequences share, against the definition in 64 bits (tests/kv_reference.py)."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
import kv_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture
def ctx(bfv):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=0)
    yield c
    c.close()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen).to(dtype)


def check(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"error is {over:.3f} of the bound"


class Shared:
    """Groups [(shared tokens, [(own tokens, new tokens), ...]), ...].  What a call may not read is NaN (pages) or -1
    (the table): first tokens of all but a group's first sequence, and pages that hold nothing else."""

    def __init__(self, bfv, ctx, groups, kv_heads, group, dim, page, dtype, layout="hnd", layers=1, layer=0, spread=1.0, seed=3,
                 width=None):
        gen = torch.Generator().manual_seed(seed)
        self.lens = [(p + own, new) for p, seqs in groups for own, new in seqs]
        cache = R.Cache(kv_heads, dim, page, dtype, [n for n, _ in self.lens], layers, layout, seed=seed, width=width)
        heads, tokens = kv_heads * group, sum(n for _, n in self.lens)
        q = randn(gen, tokens, heads + 3, dim, dtype=dtype) * spread
        self.q = q.cuda()[:, 1:1 + heads]
        self.kv_of, s = [], 0
        for p, seqs in groups:
            first = [randn(gen, p, kv_heads, dim, dtype=dtype) for _ in range(2)]
            for i, (own, _) in enumerate(seqs):
                k, v = (torch.cat([x, randn(gen, own, kv_heads, dim, dtype=dtype)]) for x in first)
                cache.put(s, k, v, layer, only=torch.arange(p + own) >= (p if i else 0))
                if i:
                    cache.table[s, :p // page] = -1
                self.kv_of.append((k, v))
                s += 1
        self.kv, self.cache = bfv.PagedKv(ctx, cache.k, cache.v), cache
        self.table, self.lengths = cache.table.cuda(), ints([n for n, _ in self.lens])
        self.starts = torch.tensor([0] + [n for _, n in self.lens]).cumsum(0).int().cuda()
        self.groups = torch.tensor([0] + [len(seqs) for _, seqs in groups]).cumsum(0).int().cuda()
        self.shared = ints([p for p, _ in groups])
        self.single = all(n == 1 for _, n in self.lens)
        self.layer, self.cpu_q = layer, q[:, 1:1 + heads]

    def run(self, **kw):
        kw.setdefault("layer", self.layer)
        if self.single:
            return self.kv.decode_shared(self.q, self.table, self.lengths, self.groups, self.shared, **kw)
        return self.kv.prompt_shared(self.q, self.starts, self.table, self.lengths, self.groups, self.shared, **kw)

    def want(self, two_terms=True, scale=None):
        out, row = [], 0
        for (length, new), (k, v) in zip(self.lens, self.kv_of):
            out.append(R.attention(self.cpu_q[row:row + new], k, v, length, 0, 0, scale or k.shape[2] ** -0.5, two_terms))
            row += new
        return [torch.cat(x) for x in zip(*out)]


def run(bfv, ctx, *a, kernels=None, scale=None, **kw):
    """kernels: those that the call has to take."""
    case = Shared(bfv, ctx, *a, **kw)
    taken = case.kv.shared_kernels(case.q, case.table, len(case.shared))
    assert kernels is None or taken == kernels
    two_terms = taken == ("rows", "rows")
    call = {} if scale is None else dict(scale=scale)
    got = case.run(**call)
    assert ctx.check() == 0
    assert torch.equal(got, case.run(**call))  # the same inputs give the same bits
    check(got, *case.want(two_terms, scale))
    return case


one = lambda *own: [(n, 1) for n in own]  # noqa: E731
DECODE = [
    # groups, kv_heads, group, dim, page, dtype, layout
    ([(1, one(0))], 1, 1, 8, 16, BF, "hnd"),                                    # nothing but the shared token
    ([(0, one(1))], 8, 2, 128, 16, BF, "hnd"),                                  # nothing shared
    ([(5, one(1, 2, 30)), (0, one(7, 0)), (100, one(1))], 2, 2, 64, 16, FP, "nhd"),
    ([(992, one(*[1 + 2 * i for i in range(16)]))], 8, 2, 128, 16, BF, "hnd"),  # answers forked from a document
    ([(1000, one(1, 40)), (16, one(3, 1, 1)), (17, one(0, 1)), (15, one(1))], 3, 5, 72, 32, FP, "gaps"),
    ([(300, one(*range(1, 41))), (77, one(2, 2))], 1, 3, 64, 16, BF, "nhd"),    # more than 32 sequences
    ([(20 + i, one(1, i)) for i in range(40)], 2, 1, 96, 16, FP, "hnd"),        # more than 32 groups
    ([(700, one(3, 100, 17))], 1, 17, 128, 64, BF, "hnd"),                      # more query heads than one unit's rows
    ([(5000, one(1, 300))], 1, 8, 128, 256, FP, "hnd"),
    ([(40, one(2000, 3000, 1)), (3000, one(1))], 2, 4, 64, 32, BF, "hnd"),      # long own parts
]
MORE = [
    # several new tokens each
    ([(64, [(5, 5), (1, 1), (9, 4), (0, 0)])], 2, 2, 64, 16, BF, "hnd"),
    ([(100, [(16, 16), (33, 33), (1, 1), (0, 1)]), (0, [(7, 7), (0, 0)]), (31, [(40, 2)])], 1, 3, 72, 32, FP, "gaps"),
    ([(513, [(20 + i, 20) for i in range(10)])], 4, 4, 128, 16, FP, "hnd"),
    ([(10, [(300, 300), (200, 17)]), (1, [(90, 90)])], 2, 2, 128, 64, BF, "nhd"),
    ([(33, [(0, 0)]), (17, [(3, 3)] * 33)], 1, 1, 96, 16, BF, "hnd"),
]
name = lambda c: "-".join(str(x).replace("torch.", "") for x in c[1:]) + "-%d" % len(c[0])  # noqa: E731


@pytest.mark.parametrize("case", DECODE, ids=name)
def test_decode_shared(bfv, ctx, case):
    groups, g, r, dim, page, dtype, layout = case
    run(bfv, ctx, groups, g, r, dim, page, dtype, layout)


@pytest.mark.parametrize("case", MORE, ids=name)
def test_prompt_shared(bfv, ctx, case):
    groups, g, r, dim, page, dtype, layout = case
    run(bfv, ctx, groups, g, r, dim, page, dtype, layout)


def repeated(own, new, count):
    return [(own, new)] * count


TILES = [
    # groups, kv_heads, group, dim, page, dtype, layout, kernels
    ([(300, one(*range(1, 131)))], 1, 2, 64, 16, BF, "nhd", ("tiles", "rows")),        # 260 rows: two units
    ([(1000, one(*range(40))), (129, one(*range(1, 40)))], 2, 8, 128, 16, BF, "hnd", ("tiles", "rows")),
    ([(17, one(*range(1, 100)))], 1, 5, 72, 32, FP, "gaps", ("tiles", "rows")),         # tokens cut between the row tiles
    ([(3000, one(*[3] * 64)), (1, one(*[1] * 64)), (128, one(*[2] * 64))], 3, 3, 128, 64, FP, "nhd", ("tiles", "rows")),
    ([(2000, one(1, 1, 1))], 1, 200, 96, 128, BF, "hnd", ("tiles", "tiles")),          # a group of 200 query heads
    ([(500, [(64, 64), (100, 80), (0, 1), (70, 70)])], 2, 2, 64, 16, BF, "hnd", ("tiles", "tiles")),
    ([(700, [(1300, 1000)]), (0, [(257, 257)]), (127, [(200, 3), (400, 333)])], 2, 3, 72, 32, FP, "gaps", ("tiles", "tiles")),
    ([(129, repeated(150, 130, 5)), (4000, repeated(129, 129, 2))], 1, 4, 128, 64, BF, "hnd", ("tiles", "tiles")),
    ([(64, [(900, 900)]), (1, repeated(300, 256, 3))], 4, 1, 128, 16, FP, "nhd", ("tiles", "tiles")),
    ([(0, [(500, 500)]), (0, [(0, 0), (300, 300)])], 1, 2, 64, 256, BF, "hnd", ("tiles", "tiles")),  # nothing shared
]


@pytest.mark.parametrize("case", TILES, ids=name)
def test_tiles(bfv, ctx, case):
    groups, g, r, dim, page, dtype, layout, kernels = case
    # (the choice goes by what a table can name)
    run(bfv, ctx, groups, g, r, dim, page, dtype, layout, kernels=kernels, width=40000 // page)
