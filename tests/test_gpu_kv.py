"""The paged key-value cache's kernels against the definition in 64 bits (tests/kv_reference.py)."""
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


def randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen).to(dtype)


def check(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"error is {over:.3f} of the bound"


def run_attention(bfv, ctx, kind, dtype, lens, kv_heads, group, dim, page, window=0, sinks=0, layout="hnd", layers=1,
                  layer=0, spread=1.0, width=None, scale=None, trim=True, seed=7):
    """lens: (length, new tokens) per sequence.  Values that no query sees are NaN in the cache."""
    gen = torch.Generator().manual_seed(seed)
    cache = R.Cache(kv_heads, dim, page, dtype, [n for n, _ in lens], layers, layout, width=width)
    heads = kv_heads * group
    tokens = sum(n for _, n in lens)
    q_all = randn(gen, tokens, heads + 3, dim, dtype=dtype) * spread
    q_dev = q_all.cuda()[:, 1:1 + heads]  # inside wider rows
    scale = scale or dim ** -0.5
    want, bound, row = [], [], 0
    for s, (length, new) in enumerate(lens):
        k, v = randn(gen, length, kv_heads, dim, dtype=dtype), randn(gen, length, kv_heads, dim, dtype=dtype)
        seen = R.visible(range(length - new, length), length, window, sinks).any(0) if new else torch.zeros(length, dtype=torch.bool)
        cache.put(s, k, v, layer, only=seen)
        if window and trim:
            cache.trim(s, length - new, window, sinks)
        q = q_all[row:row + new, 1:1 + heads]
        o, b = R.attention(q, k, v, length, window, sinks, scale, two_terms=kind == "decode")
        want.append(o)
        bound.append(b)
        row += new
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    table = cache.table.cuda()
    lengths = torch.tensor([n for n, _ in lens], dtype=torch.int32, device="cuda")
    call = dict(layer=layer, window=window, sinks=sinks, scale=scale)
    if kind == "decode":
        assert all(n == 1 for _, n in lens)
        got = kv.decode(q_dev, table, lengths, **call)
        again = kv.decode(q_dev, table, lengths, **call)
    else:
        starts = torch.tensor([0] + [n for _, n in lens], dtype=torch.int32).cumsum(0).int().cuda()
        got = kv.prompt(q_dev, starts, table, lengths, **call)
        again = kv.prompt(q_dev, starts, table, lengths, **call)
    assert ctx.check() == 0
    assert torch.equal(got, again)  # the same inputs give the same bits
    check(got, torch.cat(want), torch.cat(bound))


DECODE = [
    # dtype, lengths, kv_heads, group, dim, page, window, sinks, layout
    (BF, [1], 8, 2, 128, 16, 0, 0, "hnd"),
    (FP, [2, 1, 15, 16, 17, 63, 64, 65], 2, 1, 64, 16, 0, 0, "nhd"),
    (BF, [513], 8, 2, 128, 16, 0, 0, "hnd"),
    (FP, [129, 1, 700, 256, 255, 257], 4, 8, 128, 64, 0, 0, "hnd"),
    (BF, [333, 1000], 3, 5, 72, 32, 0, 0, "gaps"),
    (FP, [333, 90], 1, 9, 96, 128, 0, 0, "nhd"),
    (BF, [400, 1], 2, 16, 128, 16, 0, 0, "hnd"),
    (FP, [50, 700], 1, 17, 64, 16, 0, 0, "hnd"),      # more query heads than one unit holds
    (BF, [300], 1, 40, 8, 256, 0, 0, "hnd"),
    (BF, [5000], 1, 8, 128, 64, 0, 0, "hnd"),         # one unit: cluster and parts
    (FP, [20000], 1, 3, 64, 16, 0, 0, "nhd"),
    (BF, [1, 16, 17, 300, 2000, 4097], 2, 4, 64, 32, 16, 0, "hnd"),
    (FP, [1, 16, 17, 300, 2000, 4097], 2, 2, 128, 32, 100, 4, "nhd"),
    (BF, [1, 5, 300, 2000], 2, 2, 128, 16, 1, 17, "hnd"),
    (FP, [40, 900], 2, 2, 128, 16, 5000, 4, "hnd"),   # a window longer than the sequences
    (BF, [40, 900], 2, 2, 64, 16, 33, 5000, "hnd"),   # more first tokens than there are
    (BF, [0, 70, 0], 2, 2, 128, 16, 0, 0, "hnd"),     # rows without a sequence
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_decode(bfv, ctx, case):
    dtype, lens, g, r, dim, page, window, sinks, layout = case
    run_attention(bfv, ctx, "decode", dtype, [(n, 1) for n in lens], g, r, dim, page, window, sinks, layout)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_decode_large_scores(bfv, ctx, dtype):
    """Scores to about +-200: the running maximum has to carry them."""
    run_attention(bfv, ctx, "decode", dtype, [(900, 1), (37, 1)], 2, 2, 128, 16, spread=40.0)


def test_decode_other_layer_and_scale(bfv, ctx):
    run_attention(bfv, ctx, "decode", BF, [(90, 1), (300, 1)], 2, 2, 64, 16, layers=3, layer=2, scale=0.5)


def test_decode_wide_table(bfv, ctx):
    """A table far wider than the sequences: the split goes by the width, the work by the lengths."""
    run_attention(bfv, ctx, "decode", BF, [(90, 1), (3, 1)], 1, 2, 64, 16, width=5000)


PROMPT = [
    # dtype, (length, new), kv_heads, group, dim, page, window, sinks, layout
    (BF, [(1, 1)], 8, 2, 128, 16, 0, 0, "hnd"),
    (FP, [(16, 16), (5, 5), (1, 1)], 2, 2, 64, 16, 0, 0, "nhd"),
    (BF, [(512, 16)], 8, 2, 128, 16, 0, 0, "hnd"),
    (FP, [(300, 300)], 2, 1, 128, 64, 0, 0, "hnd"),
    (BF, [(300, 7), (129, 129), (1, 1), (700, 300)], 2, 3, 72, 32, 0, 0, "gaps"),
    (FP, [(257, 257), (640, 1), (128, 128)], 1, 8, 64, 128, 0, 0, "nhd"),
    (BF, [(1100, 1100)], 1, 2, 128, 256, 0, 0, "hnd"),
    (BF, [(700, 700)], 1, 2, 128, 16, 64, 4, "hnd"),
    (FP, [(1500, 600), (900, 900)], 2, 2, 64, 32, 200, 17, "nhd"),
    (BF, [(1500, 700)], 1, 4, 96, 16, 1, 0, "hnd"),
    (FP, [(800, 800)], 1, 5, 128, 16, 1, 1, "hnd"),
    (BF, [(800, 500)], 1, 1, 128, 64, 130, 300, "hnd"),
    (FP, [(900, 900)], 1, 2, 128, 16, 5000, 4, "hnd"),
    (BF, [(64, 0), (200, 200), (0, 0), (30, 2)], 2, 2, 128, 16, 0, 0, "hnd"),   # nothing new, nothing at all
    (BF, [(300, 150)], 1, 17, 64, 16, 50, 2, "hnd"),
    (FP, [(140, 140)], 1, 40, 8, 16, 0, 0, "hnd"),
    (BF, [(2100, 2100), (1, 1), (130, 40)], 1, 1, 128, 128, 0, 0, "nhd"),
    # few rows, many keys: the keys in parts
    (BF, [(5000, 300)], 1, 2, 64, 16, 0, 0, "hnd"),
    (FP, [(9000, 200), (3000, 500)], 1, 1, 128, 64, 0, 0, "gaps"),
    (BF, [(6000, 400)], 1, 3, 72, 32, 2500, 140, "nhd"),
    (FP, [(4500, 140), (30, 30)], 2, 2, 64, 128, 3000, 2, "hnd"),
    # more sequences than a warp looks through at once
    (FP, [(200 + 11 * i, 40 + i % 7) for i in range(70)], 1, 2, 64, 32, 0, 0, "hnd"),
    (BF, [(1 + 3 * i % 50, 1) for i in range(100)], 1, 4, 64, 16, 0, 0, "hnd"),
]


@pytest.mark.parametrize("case", PROMPT, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_prompt(bfv, ctx, case):
    dtype, lens, g, r, dim, page, window, sinks, layout = case
    run_attention(bfv, ctx, "prompt", dtype, lens, g, r, dim, page, window, sinks, layout)


@pytest.mark.parametrize("new", [1, 6, 500])
def test_broadcast_and_transposed_queries(bfv, ctx, new):
    """Queries with a stride of 0 over the heads or the tokens (broadcast), and with the tokens inside the
    heads."""
    gen = torch.Generator().manual_seed(4)
    cache = R.Cache(2, 64, 16, BF, [700])
    k, v = randn(gen, 700, 2, 64, dtype=BF), randn(gen, 700, 2, 64, dtype=BF)
    cache.put(0, k, v)
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([700], dtype=torch.int32, device="cuda")
    one = randn(gen, new, 1, 64, dtype=BF)
    for q in (one.cuda().expand(new, 4, 64), one[:1].cuda().expand(new, 4, 64),
              randn(gen, 4, new, 64, dtype=BF).cuda().transpose(0, 1)):
        want, bound = R.attention(q.cpu(), k, v, 700, 0, 0, 0.125, two_terms=False)
        check(kv.prompt(q, starts, cache.table.cuda(), lengths), want, bound)
        if new == 1:
            check(kv.decode(q, cache.table.cuda(), lengths), want, bound)
    assert ctx.check() == 0


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("new", [10, 600])
def test_prompt_large_scores(bfv, ctx, dtype, new):
    run_attention(bfv, ctx, "prompt", dtype, [(900, new)], 2, 2, 128, 16, spread=40.0)


def test_prompt_more_queries_than_tokens(bfv, ctx):
    """Rows before the sequence's begin see nothing: zeros."""
    for new, page in ((40, 16), (400, 64)):
        cache = R.Cache(2, 64, page, BF, [30])
        gen = torch.Generator().manual_seed(3)
        k, v = randn(gen, 30, 2, 64, dtype=BF), randn(gen, 30, 2, 64, dtype=BF)
        cache.put(0, k, v)
        q = randn(gen, new, 4, 64, dtype=BF)
        kv = bfv.PagedKv(ctx, cache.k, cache.v)
        got = kv.prompt(q.cuda(), torch.tensor([0, new], dtype=torch.int32, device="cuda"), cache.table.cuda(),
                        torch.tensor([30], dtype=torch.int32, device="cuda"))
        assert ctx.check() == 0
        assert (got[:new - 30] == 0).all()
        want, bound = R.attention(q[new - 30:], k, v, 30, 0, 0, 64 ** -0.5, two_terms=False)
        check(got[new - 30:], want, bound)


def test_infinite_and_nan_keys(bfv, ctx):
    """A visible NaN reaches its own heads and sequence, nothing else; a visible -inf score weighs 0."""
    gen = torch.Generator().manual_seed(5)
    cache = R.Cache(2, 64, 16, FP, [100, 100, 100])
    k, v = randn(gen, 100, 2, 64, dtype=FP), randn(gen, 100, 2, 64, dtype=FP)
    q = randn(gen, 3, 4, 64, dtype=FP).abs() + 0.5
    for s in range(3):
        cache.put(s, k, v)
    p, r = cache.where(1)
    cache.v[0, p[50], 0, r[50], 3] = math.nan
    p, r = cache.where(2)
    cache.k[0, p[50], :, r[50], 3] = -math.inf
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    got = kv.decode(q.cuda(), cache.table.cuda(), torch.full((3,), 100, dtype=torch.int32, device="cuda")).cpu()
    assert ctx.check() == 0
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all()
    nan = torch.isnan(got[1])
    assert nan[:2, 3].all() and nan.sum() == 2
    keep = torch.arange(100) != 50
    for h in range(4):
        o, b = R.rows(q[2:3, h], k[keep][:, h // 2], v[keep][:, h // 2], torch.ones(1, 99, dtype=torch.bool), 0.125, True)
        check(got[2:3, h], o, b)


def test_bad_tables_are_recorded_not_followed(bfv, ctx):
    """Page numbers, lengths and starts outside their range: the access is skipped and recorded."""
    cache = R.Cache(2, 64, 16, BF, [40, 40])
    gen = torch.Generator().manual_seed(5)
    for s in range(2):
        cache.put(s, randn(gen, 40, 2, 64, dtype=BF), randn(gen, 40, 2, 64, dtype=BF))
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(gen, 2, 4, 64, dtype=BF).cuda()
    good = kv.decode(q, cache.table.cuda(), dev([40, 40]))
    assert ctx.check() == 0

    def recorded():
        with pytest.raises(bfv.BfvGpuError, match="E_KV_TABLE"):
            ctx.check()
        assert ctx.check() == 0

    for bad in (-1, cache.k.shape[1], 2 ** 31 - 1, -2 ** 31):
        table = cache.table.clone()
        table[1, 1] = bad
        got = kv.decode(q, table.cuda(), dev([40, 40]))
        recorded()
        assert torch.equal(got[0], good[0])
        before, before_v = cache.k.clone(), cache.v.clone()
        kv.append(q[:, :2], q[:, 2:], None, table.cuda(), dev([5, 20]))
        recorded()
        changed = (before.view(torch.int16) != cache.k.view(torch.int16)).flatten(2).any(2)[0].nonzero().flatten().tolist()
        assert changed == [int(cache.table[0, 0])]
        cache.k.copy_(before)
        cache.v.copy_(before_v)
    for lengths in ([40, -3], [40, 10 ** 6]):
        kv.decode(q, cache.table.cuda(), dev(lengths))
        recorded()
    many = randn(gen, 300, 4, 64, dtype=BF).cuda()
    for starts in ([0, 5, 301], [0, -5, 300], [0, 400, 300]):
        kv.prompt(many, dev(starts), cache.table.cuda(), dev([40, 40]))
        recorded()


def test_pages_beyond_32_bits(bfv, ctx):
    """Offsets past 2^31 elements: a cache of 2.2 G elements, the sequence in its last pages."""
    page, heads, dim, pages = 256, 8, 128, 8600
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    k = torch.empty(pages, heads, page, dim, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    gen = torch.Generator().manual_seed(5)
    length = 300
    kk, vv = randn(gen, length, heads, dim, dtype=BF), randn(gen, length, heads, dim, dtype=BF)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
    kv = bfv.PagedKv(ctx, k, v)
    starts = torch.tensor([0, length], dtype=torch.int32, device="cuda")
    kv.append(kk.cuda(), vv.cuda(), starts, table, lengths)
    q = randn(gen, length, heads * 2, dim, dtype=BF)
    want, bound = R.attention(q, kk, vv, length, 0, 0, dim ** -0.5, two_terms=False)
    check(kv.prompt(q.cuda(), starts, table, lengths), want, bound)
    check(kv.decode(q[-1:].cuda(), table, lengths), want[-1:], bound[-1:])
    src = torch.tensor([pages - 2, pages - 1], dtype=torch.int32, device="cuda")
    kv.move(src, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), table)
    assert table.tolist() == [[1, 0]]
    check(kv.decode(q[-1:].cuda(), table, lengths), want[-1:], bound[-1:])
    assert ctx.check() == 0


# ---- pages ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["hnd", "nhd", "gaps"])
@pytest.mark.parametrize("dtype,source", [(BF, BF), (FP, FP), (BF, torch.float32), (FP, torch.float32)])
def test_append(bfv, ctx, layout, dtype, source):
    gen = torch.Generator().manual_seed(9)
    lens = [(40, 40), (17, 1), (0, 0), (100, 30), (64, 0), (16, 16)]
    for heads, dim, page in ((2, 64, 16), (3, 72, 32), (8, 128, 16), (1, 8, 256)):
        cache = R.Cache(heads, dim, page, dtype, [n for n, _ in lens], layers=2, layout=layout)
        tokens = sum(n for _, n in lens)
        row = (randn(gen, tokens, 3 * heads + 1, dim) * 100).to(source).cuda()
        k_new, v_new = row[:, heads:2 * heads], row[:, 2 * heads:3 * heads]
        want_k, want_v = cache.k.clone(), cache.v.clone()
        at = 0
        for s, (length, new) in enumerate(lens):
            for i in range(new):
                p = length - new + i
                pg, r = int(cache.table[s, p // page]), p % page
                want_k[1, pg, :, r] = k_new[at].to(dtype)
                want_v[1, pg, :, r] = v_new[at].to(dtype)
                at += 1
        starts = torch.tensor([0] + [n for _, n in lens]).cumsum(0).int().cuda()
        lengths = torch.tensor([n for n, _ in lens], dtype=torch.int32, device="cuda")
        kv = bfv.PagedKv(ctx, cache.k, cache.v)
        kv.append(k_new, v_new, starts, cache.table.cuda(), lengths, layer=1)
        assert ctx.check() == 0
        same = lambda a, b: torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))  # noqa: E731
        assert same(cache.k, want_k) and same(cache.v, want_v)


def test_append_one_token_each(bfv, ctx):
    cache = R.Cache(2, 64, 16, BF, [1, 16, 17, 40])
    gen = torch.Generator().manual_seed(9)
    k, v = randn(gen, 4, 2, 64, dtype=BF).cuda(), randn(gen, 4, 2, 64, dtype=BF).cuda()
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    kv.append(k, v, None, cache.table.cuda(), torch.tensor([1, 16, 17, 40], dtype=torch.int32, device="cuda"))
    assert ctx.check() == 0
    for s, n in enumerate([1, 16, 17, 40]):
        p, r = cache.where(s)
        assert torch.equal(cache.k[0, p[-1], :, r[-1]], k[s]) and torch.equal(cache.v[0, p[-1], :, r[-1]], v[s])
    assert torch.isfinite(cache.k).sum() == 4 * 2 * 64


def _fill(cache, gen):
    for x in (cache.k, cache.v):
        x.copy_(torch.randn(x.shape, generator=gen).to(x.dtype))


@pytest.mark.parametrize("layout", ["hnd", "nhd", "gaps"])
@pytest.mark.parametrize("length", [1, 16, 37, 64])
def test_fork(bfv, ctx, layout, length):
    gen = torch.Generator().manual_seed(9)
    cache = R.Cache(3, 72, 16, FP, [length, 5, 0, 0, 0], layers=3, layout=layout, spare=6, width=5)
    _fill(cache, gen)
    want_k, want_v, table = cache.k.clone(), cache.v.clone(), cache.table.clone()
    fresh = cache.spare[:3].clone()
    last = length // 16
    for c in range(3):
        table[2 + c] = table[0]
        if length % 16:
            table[2 + c, last] = fresh[c]
            want_k[:, fresh[c]] = want_k[:, table[0, last]]
            want_v[:, fresh[c]] = want_v[:, table[0, last]]
        else:
            fresh[c] = -1
    dev = cache.table.cuda()
    lengths = torch.tensor([length, 5, 0, 0, 0], dtype=torch.int32, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bfv.PagedKv(ctx, cache.k, cache.v).fork(ints([0, 0, 0]), ints([2, 3, 4]), fresh.cuda(), dev, lengths)
    assert ctx.check() == 0
    assert torch.equal(dev.cpu(), table) and lengths.tolist() == [length, 5, length, length, length]
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


@pytest.mark.parametrize("layout", ["hnd", "nhd", "gaps"])
def test_move(bfv, ctx, layout):
    gen = torch.Generator().manual_seed(9)
    cache = R.Cache(2, 64, 32, BF, [100, 33, 64, 200], layers=2, layout=layout, spare=9)
    _fill(cache, gen)
    want_k, want_v, table = cache.k.clone(), cache.v.clone(), cache.table.clone()
    used = table[table >= 0]
    src = used[::2].sort().values
    dst = cache.spare[:len(src)].clone()
    assert len(src) == len(dst)
    for a, b in zip(src.tolist(), dst.tolist()):
        want_k[:, b], want_v[:, b] = want_k[:, a], want_v[:, a]
        table[cache.table == a] = b
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    dev = cache.table.cuda()
    kv.move(src.cuda(), dst.cuda(), dev)
    assert ctx.check() == 0
    assert torch.equal(dev.cpu(), table)
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
    kv.move(src[:0].cuda(), dst[:0].cuda(), dev)  # nothing to do
    assert torch.equal(dev.cpu(), table)


def test_move_and_fork_reject_bad_numbers(bfv, ctx):
    cache = R.Cache(2, 64, 16, BF, [40, 0])
    gen = torch.Generator().manual_seed(9)
    _fill(cache, gen)
    before = cache.k.clone()
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = cache.k.shape[1]
    for src, dst in (([-1], [0]), ([pages], [0]), ([0], [pages]), ([0], [-1])):
        table = cache.table.cuda()
        kv.move(ints(src), ints(dst), table)
        with pytest.raises(bfv.BfvGpuError, match="E_KV_TABLE"):
            ctx.check()
        assert torch.equal(table.cpu(), cache.table)
    for parent, child, fresh in ((2, 1, 0), (-1, 1, 0), (0, 2, 0), (0, 0, 0), (0, 1, pages), (0, 1, -1)):
        table, lengths = cache.table.cuda(), ints([40, 0])
        kv.fork(ints([parent]), ints([child]), ints([fresh]), table, lengths)
        with pytest.raises(bfv.BfvGpuError, match="E_KV_TABLE"):
            ctx.check()
        assert torch.equal(table.cpu(), cache.table) and lengths.tolist() == [40, 0]
    assert torch.equal(before, cache.k)


def test_refused_tensors(bfv, ctx):
    """What the calls refuse before any launch: types, shapes, strides, devices, numbers out of 32 bits."""
    cache = R.Cache(2, 64, 16, BF, [40, 9])
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    dev = dict(device="cuda")
    table, lengths = cache.table.cuda(), torch.tensor([40, 9], dtype=torch.int32, **dev)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, **dev)
    q, k = torch.zeros(2, 4, 64, dtype=BF, **dev), torch.zeros(2, 2, 64, dtype=BF, **dev)
    ids = torch.tensor([0, 1], dtype=torch.int32, **dev)
    wide = torch.zeros(2, 4, 128, dtype=BF, **dev)
    refused = [
        lambda: kv.decode(q[:1], table, lengths), lambda: kv.decode(q[0], table, lengths),
        lambda: kv.decode(wide, table, lengths), lambda: kv.decode(wide[..., ::2], table, lengths),
        lambda: kv.decode(q.cpu(), table, lengths), lambda: kv.decode(q.half(), table, lengths),
        lambda: kv.decode(q, table.cpu(), lengths), lambda: kv.decode(q, table.long(), lengths),
        lambda: kv.decode(q, table.t(), lengths), lambda: kv.decode(q, table[0], lengths),
        lambda: kv.decode(q, table, lengths[:1]), lambda: kv.decode(q, table, lengths.float()),
        lambda: kv.decode(q, table, lengths, layer=1), lambda: kv.decode(q, table, lengths, window=-1),
        lambda: kv.decode(q, table, lengths, scale=-1.0), lambda: kv.decode(q[:, :3], table, lengths),
        lambda: kv.decode(q, table, lengths, out=q[:1]), lambda: kv.decode(q, table, lengths, out=q.half()),
        lambda: kv.decode(q, table, lengths, out=wide[..., :64]),
        lambda: kv.prompt(q, starts[:2], table, lengths), lambda: kv.prompt(q, starts.cpu(), table, lengths),
        lambda: kv.append(k, k.half(), starts, table, lengths), lambda: kv.append(k.half(), k.half(), starts, table, lengths),
        lambda: kv.append(k, k[:1], starts, table, lengths), lambda: kv.append(q, q, starts, table, lengths),
        lambda: kv.append(k, k, starts[:2], table, lengths),
        lambda: kv.fork(ids, ids[:1], ids, table, lengths), lambda: kv.fork(ids, ids, ids.long(), table, lengths),
        lambda: kv.fork(ids, ids, ids, table, lengths[:1]),
        lambda: kv.move(ids, ids[:1], table), lambda: kv.move(ids.cpu(), ids, table), lambda: kv.move(ids, ids, lengths),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError, match="E_KV_"):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(OverflowError):
        kv.decode(q, table, lengths, window=1 << 40)
    assert ctx.check() == 0
    out = torch.empty_like(q)
    assert kv.decode(q, table, lengths, out=out) is out


@pytest.mark.parametrize("dim,window,sinks", [(112, 0, 0), (64, 0, 0), (128, 3, 2)])
def test_rows_past_the_last_change_nothing(bfv, ctx, dim, window, sinks):
    """Many prompts of odd lengths whose query heads do not fill a block's rows, with scores that move the reference
    exponent often: what the unused rows held before must not show in the others, not even in the last bit."""
    lens = [(17, 16), (257, 257), (127, 1), (200, 200), (256, 1), (17, 17), (128, 16), (255, 255), (0, 0), (1, 1), (511, 128),
            (300, 33), (640, 2), (63, 0), (31, 31), (257, 3), (128, 100), (127, 127), (127, 64), (64, 64), (257, 128),
            (256, 256), (16, 16), (129, 0), (255, 16), (300, 100), (31, 31), (129, 64), (127, 33)]
    run_attention(bfv, ctx, "prompt", BF, lens, 3, 9, dim, 16, window, sinks, spread=4.0)


# ---- streams, graphs, the whole cache -------------------------------------------------------------
def test_other_stream_and_graph(bfv, ctx):
    """The calls on a side stream, and captured in a graph and replayed on new values, give the bits of
    the calls on the default stream."""
    gen = torch.Generator().manual_seed(11)
    cache = R.Cache(2, 128, 16, BF, [700, 90, 5])
    _fill(cache, gen)
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    table = cache.table.cuda()
    lengths = torch.tensor([700, 90, 5], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    q = randn(gen, 3, 4, 128, dtype=BF).cuda()
    want = kv.decode(q, table, lengths)
    want_p = kv.prompt(q, starts, table, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv.decode(q, table, lengths)
    handle = kv.decode(q, table, lengths, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(handle, want)
    out, out_p, q_in = torch.empty_like(want), torch.empty_like(want), torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.append(q_in[:, :2], q_in[:, 2:], None, table, lengths)
        kv.decode(q_in, table, lengths, out=out)
        kv.prompt(q_in, starts, table, lengths, out=out_p)
    k0, v0 = cache.k.clone(), cache.v.clone()
    for scale in (1.0, 2.0):
        q_in.copy_(q * scale)
        graph.replay()
        torch.cuda.synchronize()
        k1, v1 = cache.k.clone(), cache.v.clone()
        cache.k.copy_(k0)
        cache.v.copy_(v0)
        kv.append(q_in[:, :2], q_in[:, 2:], None, table, lengths)
        assert torch.equal(k1, cache.k) and torch.equal(v1, cache.v)
        assert torch.equal(out, kv.decode(q_in, table, lengths))
        assert torch.equal(out_p, kv.prompt(q_in, starts, table, lengths))
    assert ctx.check() == 0


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_cache_of_forked_sequences(bfv, ctx, window, sinks):
    """A session: prompts, forks, steps, ends, trims and compaction, against a history kept in a list."""
    gen = torch.Generator().manual_seed(13)
    heads, group, dim, layers = 2, 2, 64, 2
    cache = bfv.KvCache(ctx, pages=60, heads=heads, dim=dim, layers=layers, page_tokens=16, sequences=6, tokens=400,
                        dtype=FP)
    history = {}

    def step(counts):
        cache.extend(counts)
        tokens = sum(counts.values())
        for layer in range(layers):
            k, v = randn(gen, tokens, heads, dim, dtype=FP), randn(gen, tokens, heads, dim, dtype=FP)
            q = randn(gen, tokens, heads * group, dim, dtype=FP)
            cache.append(k.cuda(), v.cuda(), layer)
            got = cache.attend(q.cuda(), layer, window, sinks)
            at = 0
            for row in sorted(counts):
                n = counts[row]
                hk, hv = history[row][layer]
                history[row][layer] = hk, hv = torch.cat([hk, k[at:at + n]]), torch.cat([hv, v[at:at + n]])
                want, bound = R.attention(q[at:at + n], hk, hv, len(hk), window, sinks, dim ** -0.5, two_terms=False)
                check(got[at:at + n], want, bound)
                at += n
        assert ctx.check() == 0

    def begin():
        row = cache.open()
        history[row] = [(torch.zeros(0, heads, dim, dtype=FP),) * 2 for _ in range(layers)]
        return row

    a, b = begin(), begin()
    step({a: 37, b: 20})
    kids = cache.fork(a, 3)
    for c in kids:
        history[c] = list(history[a])
    step({a: 1, kids[0]: 1, kids[1]: 5, kids[2]: 16, b: 1})
    cache.free(a)
    del history[a]
    step({r: 1 for r in history})
    if window:
        step({r: 60 for r in history})
        assert cache.trim(window, sinks) > 0
    assert cache.compact() > 0
    assert (cache.book.refs[:(cache.book.refs > 0).sum()] > 0).all()
    c = begin()
    step({**{r: 1 for r in history}, c: 30})
    cache.free(kids[1])
    del history[kids[1]]
    again = cache.fork(kids[0], 1)[0]
    history[again] = list(history[kids[0]])
    rest = begin()
    step({r: 2 if r == rest else 1 for r in history})
    step({r: 1 for r in history})  # every row one token: the single-token form
    assert torch.equal(cache.table.cpu(), torch.from_numpy(cache.book.table))
    assert torch.equal(cache.lengths.cpu(), torch.from_numpy(cache.book.lengths))


@pytest.mark.parametrize("layout", ["hnd", "nhd", "gaps"])
@pytest.mark.parametrize("heads,dim", [(3, 40), (1, 8), (5, 128)])
def test_fork_and_move_of_large_pages(bfv, ctx, layout, heads, dim):
    """Pages of several shares of the copy kernels, the last one partly filled, and of less than one."""
    cache = R.Cache(heads, dim, 256, BF, [300, 0], layers=2, layout=layout, spare=3, width=2)
    _fill(cache, torch.Generator().manual_seed(9))
    want_k, want_v = cache.k.clone(), cache.v.clone()
    fresh, to = cache.spare[:1].clone(), cache.spare[1:2].clone()
    first, last = cache.table[0, :1].clone(), cache.table[0, 1:2].clone()
    for x in (want_k, want_v):
        x[:, fresh.long()] = x[:, last.long()]
        x[:, to.long()] = x[:, first.long()]
    table, lengths = cache.table.cuda(), torch.tensor([300, 0], dtype=torch.int32, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kv = bfv.PagedKv(ctx, cache.k, cache.v)
    kv.fork(ints([0]), ints([1]), fresh.cuda(), table, lengths)
    kv.move(first.cuda(), to.cuda(), table)
    assert ctx.check() == 0
    assert table.tolist() == [[int(to), int(last)], [int(to), int(fresh)]] and lengths.tolist() == [300, 300]
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
