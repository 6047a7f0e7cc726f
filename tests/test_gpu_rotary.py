"""Rotary positions and the append that applies them, against the definition (tests/rotary_reference.py)."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
import kv_reference as R  # noqa: E402
import rotary_reference as RR  # noqa: E402

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def memory_given_back():
    """What torch has cached goes back, so that the tests after these allocate as without them (calls on a context's own
    stream are not ordered after torch's, which an allocation from the driver hides)."""
    yield
    if torch.cuda.is_available():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()


@pytest.fixture
def ctx(bfv):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=0)
    yield c
    c.close()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen).to(dtype)


def check(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"error is {over:.3f} of the bound"


APPLY = [
    # dtype, tokens, heads, dim, dims, layout, norm, inverse, how the rows lie
    (BF, 1, 1, 8, 8, "half", False, False, "dense"),
    (FP, 1, 1, 8, 4, "interleaved", True, False, "dense"),
    (F32, 3, 5, 128, 128, "half", True, False, "joint"),
    (BF, 7, 24, 128, 128, "half", False, False, "joint"),
    (BF, 33, 16, 128, 64, "interleaved", True, False, "heads outside"),
    (FP, 65, 3, 72, 72, "half", True, False, "joint"),
    (FP, 130, 2, 72, 36, "half", False, True, "dense"),        # runs of two
    (F32, 9, 7, 80, 20, "half", True, False, "joint"),
    (F32, 20, 2, 72, 68, "interleaved", False, True, "heads outside"),
    (BF, 50, 9, 96, 24, "half", True, False, "dense"),
    (FP, 2500, 12, 64, 64, "half", False, True, "joint"),      # more tokens than warps
    (BF, 2500, 5, 96, 96, "interleaved", True, False, "joint"),
    (F32, 3000, 1, 128, 4, "half", False, True, "dense"),
    (BF, 10, 65, 128, 124, "half", True, False, "same token"),
]


@pytest.mark.parametrize("case", APPLY, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_apply(bfv, ctx, case):
    dtype, tokens, heads, dim, dims, layout, with_norm, inverse, lie = case
    gen = torch.Generator().manual_seed(5)
    if lie == "joint":
        whole = randn(gen, tokens, heads + 3, dim, dtype=dtype)
        x, dev = whole[:, 2:2 + heads], whole.cuda()[:, 2:2 + heads]
    elif lie == "heads outside":
        whole = randn(gen, heads, tokens, dim, dtype=dtype)
        x, dev = whole.transpose(0, 1), whole.cuda().transpose(0, 1)
    elif lie == "same token":  # a broadcast axis
        whole = randn(gen, 1, heads, dim, dtype=dtype)
        x, dev = whole.expand(tokens, heads, dim), whole.cuda().expand(tokens, heads, dim)
    else:
        x = randn(gen, tokens, heads, dim, dtype=dtype)
        dev = x.cuda()
    norm = 1 + 0.3 * randn(gen, dim) if with_norm else None
    positions = torch.randint(0, 1 << 17, (tokens,), generator=gen)
    positions[0] = 0
    rotary = bfv.Rotary(ctx, dims, base=1e6, layout=layout, scaling="yarn" if dims >= 8 else "linear", factor=4.0)
    want, bound = RR.rotate(x, positions, rotary.radians, rotary.scale, layout, norm, 1e-5, inverse)
    call = dict(norm=None if norm is None else norm.cuda(), eps=1e-5, inverse=inverse)
    got = rotary.apply(dev, positions.int().cuda(), **call)
    assert got.is_contiguous() and got.dtype == dtype
    check(got, want, bound)
    assert torch.equal(got, rotary.apply(dev, positions.int().cuda(), **call))
    if lie != "same token":  # in place, and into rows that lie otherwise
        out = torch.full((tokens, heads + 1, dim + 8), math.nan, dtype=dtype, device="cuda")
        assert rotary.apply(dev, positions.int().cuda(), out=out[:, 1:, 8:], **call).data_ptr() == out[:, 1:, 8:].data_ptr()
        assert torch.equal(out[:, 1:, 8:], got) and out[:, 0].isnan().all() and out[:, :, :8].isnan().all()
        assert rotary.apply(dev, positions.int().cuda(), out=dev, **call) is dev
        assert torch.equal(dev, got)
    assert ctx.check() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_and_negative_positions(bfv, ctx, layout):
    gen = torch.Generator().manual_seed(6)
    at = [0, 1, -1, -5, 131071, (1 << 24) + 1, (1 << 30) - 1, (1 << 31) - 1, -(1 << 31)]
    x = randn(gen, len(at), 3, 64)
    rotary = bfv.Rotary(ctx, 64, base=1e4, layout=layout)
    want, bound = RR.rotate(x, at, rotary.radians, 1.0, layout)
    check(rotary.apply(x.cuda(), ints(at)), want, bound)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient(bfv, ctx, layout):
    """The rotation back against the formula (in test_apply) and against differences: for a linear call the difference of
    two results, weighted by g, is the gradient's product with the difference of the arguments."""
    gen = torch.Generator().manual_seed(7)
    tokens, heads, dim = 40, 3, 96
    rotary = bfv.Rotary(ctx, 48, layout=layout, scaling="yarn", factor=2.0)
    x, d, g = (randn(gen, tokens, heads, dim).cuda() for _ in range(3))
    at = ints(list(range(100, 100 + tokens)))
    moved = rotary.apply(x + d, at).double() - rotary.apply(x, at).double()
    back = rotary.apply(g, at, inverse=True).double()
    a, b = (g.double() * moved).sum((1, 2)), (back * d.double()).sum((1, 2))
    # a result is off by 9 2^-24 of its pair's size at most, which is twice the scale and the largest argument; the sum
    # x + d by 2^-24 of itself
    X, D, G = (t.abs().max().item() for t in (x, d, g))
    sums = [t.abs().double().sum((1, 2)) for t in (g, d)]
    bound = 2.0 ** -24 * rotary.scale * (sums[0] * (18 * (X + D) + 18 * X + 2 * (X + D)) + sums[1] * 18 * G)
    assert ((a - b).abs() <= bound).all()
    assert a.abs().max() > 1.0


def test_values_that_are_not_finite_stay_in_their_pairs(bfv, ctx):
    for layout in ("half", "interleaved"):
        for dims, dim in ((64, 128), (36, 72)):
            x = torch.ones(4, 3, dim, device="cuda")
            x[1, 1, dims] = math.nan        # of the rest
            x[2, 2, dims + 1] = math.inf
            x[3, 0, 0] = math.nan           # of a pair
            rotary = bfv.Rotary(ctx, dims, layout=layout)
            y = rotary.apply(x, ints([3, 4, 5, 6]))
            other = torch.zeros(4, 3, dim, dtype=torch.bool, device="cuda")
            other[1, 1, dims] = other[2, 2, dims + 1] = other[3, 0, 0] = True
            other[3, 0, dims // 2 if layout == "half" else 1] = True
            assert torch.equal(~y.isfinite(), other)
            assert y[2, 2, dims + 1] == math.inf


def test_sizes_without_elements(bfv, ctx):
    rotary = bfv.Rotary(ctx, 64)
    for shape in ((0, 4, 64), (4, 0, 64)):
        x = torch.zeros(*shape, device="cuda")
        assert rotary.apply(x, ints([0] * shape[0])).shape == shape


def test_apply_refusals(bfv, ctx):
    rotary, x, at = bfv.Rotary(ctx, 64), torch.zeros(4, 2, 64, device="cuda"), ints([0, 1, 2, 3])
    norm = torch.ones(64, device="cuda")
    bad = [
        dict(x=x.cpu()), dict(x=x[0]), dict(x=x.double()), dict(x=x.transpose(1, 2)), dict(positions=at[:3]),
        dict(positions=at.long()), dict(positions=at.cpu()), dict(norm=norm[:32]), dict(norm=norm.bfloat16()),
        dict(norm=norm.cpu()), dict(norm=norm, inverse=True), dict(out=x[:3]), dict(out=x.bfloat16()),
        dict(out=torch.zeros(1, 2, 64, device="cuda").expand(4, 2, 64)), dict(eps=-1.0), dict(x=x[..., 2:34]), dict(x=x[..., :32]),
        dict(x=torch.zeros(4, 2, 136, device="cuda")),
    ]
    for kw in bad:
        with pytest.raises(ValueError, match="E_ROTARY"):
            rotary.apply(**{**dict(x=x, positions=at), **kw})
    wide = torch.zeros(9, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="E_ROTARY_OVERLAP"):  # rows that others still have to read
        rotary.apply(wide[:4], at, out=wide[1:5])
    with pytest.raises(TypeError):
        rotary.apply([1.0], at)
    ctx.close()
    with pytest.raises(bfv.BfvGpuInvalidArgument, match="E_BFVGPU_ARGUMENT"):
        rotary.apply(x, at)


APPEND = [
    # dtype, source, (length, new), kv_heads, q_heads, dim, page, dims, layout, q_norm, k_norm, pages' layout
    (BF, BF, [(1, 1)], 8, 16, 128, 16, 128, "half", True, True, "hnd"),
    (BF, F32, [(17, 1), (1, 1), (16, 1), (900, 1)], 8, 16, 128, 16, 128, "half", True, True, "hnd"),
    (FP, FP, [(40, 40), (5, 3), (7, 0), (300, 257)], 2, 6, 64, 32, 32, "interleaved", False, False, "nhd"),
    (FP, F32, [(40, 40), (5, 3), (7, 0), (300, 257)], 3, 0, 72, 64, 36, "half", False, True, "gaps"),
    (BF, BF, [(100, 37), (64, 64)], 1, 8, 96, 128, 96, "half", True, False, "hnd"),
    (BF, F32, [(2000, 1999), (700, 700)], 4, 4, 80, 16, 20, "half", True, True, "nhd"),
    (FP, FP, [(9, 9)] * 70, 1, 1, 8, 16, 8, "interleaved", True, True, "hnd"),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:100])
def test_append_rotary(bfv, ctx, case):
    dtype, source, lens, g, h, dim, page, dims, layout, with_q_norm, with_k_norm, lie = case
    gen = torch.Generator().manual_seed(8)
    cache = R.Cache(g, dim, page, dtype, [n for n, _ in lens], layers=2, layout=lie)
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    rotary = bfv.Rotary(ctx, dims, layout=layout)
    tokens = sum(n for _, n in lens)
    row = randn(gen, tokens, h + 2 * g, dim, dtype=source)
    dev = row.cuda()
    q_norm, k_norm = (1 + 0.3 * randn(gen, dim) if on else None for on in (with_q_norm and h, with_k_norm))
    single = all(n == 1 for _, n in lens)
    starts = torch.tensor([0] + [n for _, n in lens]).cumsum(0).int().cuda()
    lengths = ints([n for n, _ in lens])
    up = lambda w: None if w is None else w.cuda()  # noqa: E731
    got = kv.append_rotary(dev[:, h:h + g], dev[:, h + g:], rotary, None if single else starts, cache.table.cuda(), lengths,
                           q=dev[:, :h] if h else None, q_norm=up(q_norm), k_norm=up(k_norm), layer=1)
    assert ctx.check() == 0
    at = torch.cat([torch.arange(n - new, n) for n, new in lens])
    if h:
        assert got.shape == (tokens, h, dim) and got.dtype == dtype
        check(got, *RR.rotate(row[:, :h], at, rotary.radians, 1.0, layout, q_norm, dtype=dtype))
    else:
        assert got is None
    keys, bound = RR.rotate(row[:, h:h + g], at, rotary.radians, 1.0, layout, k_norm, dtype=dtype)
    written = torch.zeros(cache.k.shape[1:4], dtype=torch.bool)
    first = 0
    for s, (n, new) in enumerate(lens):
        pages, rows = (x[n - new:] for x in cache.where(s))
        written[pages, :, rows] = True
        check(cache.k[1].cpu()[pages, :, rows], keys[first:first + new], bound[first:first + new])
        assert torch.equal(cache.v[1].cpu()[pages, :, rows], row[first:first + new, h + g:].to(dtype))
        first += new
    for x in (cache.k, cache.v):  # nothing else
        assert x[0].isnan().all() and x[1].cpu()[~written].isnan().all()


def test_the_same_as_rotating_and_appending(bfv, ctx):
    """Both calls round once, from the same 32-bit numbers (without a norm, whose sum goes by the lanes of a row)."""
    gen = torch.Generator().manual_seed(9)
    lens, g, h, dim = [(300, 200), (64, 64)], 2, 6, 128
    a, b = (R.Cache(g, dim, 32, BF, [n for n, _ in lens]) for _ in range(2))
    rotary = bfv.Rotary(ctx, 128, base=1e6, scaling="ntk", factor=2.0)
    row = randn(gen, 264, h + 2 * g, dim, dtype=BF).cuda()
    table, lengths, starts = a.table.cuda(), ints([300, 64]), ints([0, 200, 264])
    q = bfv.PagedKv(ctx, a.k, a.v).append_rotary(row[:, h:h + g], row[:, h + g:], rotary, starts, table, lengths, q=row[:, :h])
    at = ints(list(range(100, 300)) + list(range(64)))
    both = rotary.apply(row[:, :h + g], at)
    bfv.PagedKv(ctx, b.k, b.v).append(both[:, h:].contiguous(), row[:, h + g:].contiguous(), starts, table, lengths)
    assert torch.equal(q, both[:, :h])
    assert torch.equal(a.k.nan_to_num(7.0), b.k.nan_to_num(7.0)) and torch.equal(a.v.nan_to_num(7.0), b.v.nan_to_num(7.0))


def test_queries_in_place(bfv, ctx):
    cache = R.Cache(2, 64, 16, BF, [30, 20])
    kv, rotary = bfv.PagedKv(ctx, cache.k, cache.v), bfv.Rotary(ctx, 64)
    gen = torch.Generator().manual_seed(10)
    q, k, v = (randn(gen, 2, n, 64, dtype=BF).cuda() for n in (4, 2, 2))
    table, lengths = cache.table.cuda(), ints([30, 20])
    want = kv.append_rotary(k, v, rotary, None, table, lengths, q=q)
    assert kv.append_rotary(k, v, rotary, None, table, lengths, q=q, out=q) is q and torch.equal(q, want)
    # out may be neither over the rows that are read nor over the pages
    both, wide = torch.zeros(3, 4, 64, dtype=BF, device="cuda"), torch.zeros(2, 8, 64, dtype=BF, device="cuda")
    over = wide.view(-1)[:512].view(2, 4, 64)
    for kw in (dict(q=both[:2], out=both[1:]), dict(q=q, out=cache.k.view(-1)[:512].view(2, 4, 64)),
               dict(q=q, k_new=wide[:, :2], v_new=wide[:, 6:], out=over), dict(q=q, k_new=wide[:, 6:], v_new=wide[:, 2:4], out=over)):
        with pytest.raises(ValueError, match="E_KV_OVERLAP"):
            kv.append_rotary(**{**dict(k_new=k, v_new=v, rotary=rotary, starts=None, table=table, lengths=lengths), **kw})


def test_bad_numbers_on_the_device_are_recorded(bfv, ctx):
    """Nothing is written for a token whose sequence or page is outside its range, nor its queries."""
    cache = R.Cache(2, 64, 16, BF, [40, 9])
    kv, rotary = bfv.PagedKv(ctx, cache.k, cache.v), bfv.Rotary(ctx, 64)
    table = cache.table.cuda()
    row = torch.ones(12, 8, 64, dtype=BF, device="cuda")

    def run(table, lengths, starts):
        out = torch.full((12, 4, 64), 5.0, dtype=BF, device="cuda")
        kv.append_rotary(row[:, 4:6], row[:, 6:], rotary, ints(starts), table, ints(lengths), q=row[:, :4], out=out)
        with pytest.raises(bfv.BfvGpuError, match="E_KV_TABLE"):
            ctx.check()
        return out

    bad = table.clone()
    bad[0, 2] = cache.k.shape[1]
    assert (run(bad, [40, 9], [0, 8, 12])[:8] == 5.0).all()
    bad[0, 2] = -1
    assert (run(bad, [40, 9], [0, 8, 12])[:8] == 5.0).all()
    assert (run(table, [3, 9], [0, 8, 12])[:5] == 5.0).all()            # five tokens before the first position
    assert (run(table, [-3, 9], [0, 8, 12])[:8] == 5.0).all()
    assert (run(table, [40, 9], [2, 8, 12])[:2] == 5.0).all()           # tokens of no sequence
    assert (run(table, [40, 9], [0, 8, 10])[10:] == 5.0).all()
    run(table, [1 << 30, 9], [0, 8, 12])
    assert ctx.check() == 0


def test_append_refusals(bfv, ctx):
    cache = R.Cache(2, 64, 16, BF, [40, 9])
    kv, rotary = bfv.PagedKv(ctx, cache.k, cache.v), bfv.Rotary(ctx, 64)
    row = torch.ones(2, 8, 64, dtype=BF, device="cuda")
    norm = torch.ones(64, device="cuda")
    good = dict(k_new=row[:, 4:6], v_new=row[:, 6:], rotary=rotary, starts=None, table=cache.table.cuda(), lengths=ints([40, 9]))
    bad = [
        dict(k_new=row[:, 4:7]), dict(v_new=row[:, 6:].float()), dict(q=row[:1, :4]), dict(q=row[:, :4].float()),
        dict(q=row[:, :4, :32]), dict(q_norm=norm), dict(out=row[:, :4]), dict(q=row[:, :4], q_norm=norm[:8]), dict(k_norm=norm.half()),
        dict(q=row[:, :4], out=torch.ones(2, 4, 64, device="cuda")), dict(q=row[:, :4], out=row[:, :4]), dict(starts=ints([0, 2])),
        dict(rotary=bfv.Rotary(ctx, 68)), dict(eps=math.nan), dict(layer=1), dict(table=cache.table), dict(lengths=ints([40])),
    ]
    for kw in bad:
        with pytest.raises(ValueError, match="E_KV|E_ROTARY"):
            kv.append_rotary(**{**good, **kw})
    assert kv.append_rotary(**good) is None


def test_streams_and_graphs(bfv, ctx):
    """A captured step replays with new lengths, tables and rows; a named stream keeps what it uses."""
    gen = torch.Generator().manual_seed(11)
    cache = R.Cache(2, 128, 16, BF, [60, 60])
    kv, rotary = bfv.PagedKv(ctx, cache.k, cache.v), bfv.Rotary(ctx, 128)
    row = randn(gen, 2, 8, 128).cuda()
    table, lengths = cache.table.cuda(), ints([1, 1])
    call = lambda **kw: kv.append_rotary(row[:, 4:6], row[:, 6:], rotary, None, table, lengths, q=row[:, :4], **kw)  # noqa: E731
    call()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = call()
        x = rotary.apply(row, lengths)
    for step in (3, 17, 59):
        lengths.fill_(step)
        row.copy_(randn(gen, 2, 8, 128))
        graph.replay()
        q, k, whole = out.clone(), cache.k.clone(), x.clone()
        assert torch.equal(whole, rotary.apply(row, lengths))
        assert torch.equal(q, call()) and torch.equal(k.nan_to_num(9.0), cache.k.nan_to_num(9.0))
    side.wait_stream(torch.cuda.current_stream())
    on_side = call(stream=side.cuda_stream)
    also = rotary.apply(row, lengths, stream=side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, call()) and torch.equal(also, rotary.apply(row, lengths))
    assert ctx.check() == 0
