"""The calls of PagedKv on the GPU: contexts, streams, strides and starts that need care."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import kv_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture
def ctx(bfv):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=0)
    yield c
    c.close()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, *shape, dtype=BF):
    return torch.randn(*shape, generator=gen).to(dtype)


def filled(bfv, ctx, lengths, heads=2, dim=64, page=16, dtype=BF, seed=3, **kw):
    """(PagedKv, its pages, table, lengths, [(k, v)] on the CPU)."""
    gen = torch.Generator().manual_seed(seed)
    cache = R.Cache(heads, dim, page, dtype, lengths, **kw)
    held = [(randn(gen, n, heads, dim, dtype=dtype), randn(gen, n, heads, dim, dtype=dtype)) for n in lengths]
    for s, (k, v) in enumerate(held):
        cache.put(s, k, v)
    return bfv.PagedKv(ctx, cache.k, cache.v), cache, cache.table.cuda(), ints(lengths), held


def check(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max().item()
    assert over <= 1.0, f"error is {over:.3f} of the bound"


def test_a_closed_context_is_refused(bfv, ctx):
    kv, cache, table, lengths, _ = filled(bfv, ctx, [40, 9])
    q = torch.zeros(2, 4, 64, dtype=BF, device="cuda")
    one = ints([0])
    kv.decode(q, table, lengths)
    assert ctx.check() == 0
    ctx.close()
    for call in (lambda: kv.append(q[:, :2], q[:, 2:], None, table, lengths), lambda: kv.decode(q, table, lengths),
                 lambda: kv.prompt(q, ints([0, 1, 2]), table, lengths), lambda: kv.fork(one, one, one, table, lengths),
                 lambda: kv.move(one, one, table)):
        with pytest.raises(bfv.BfvGpuInvalidArgument, match="E_BFVGPU_ARGUMENT"):
            call()


@pytest.mark.parametrize("dim", [8, 40, 56, 64, 72, 88, 104, 120, 128])
@pytest.mark.parametrize("seqs,group", [(1, 1), (1, 16), (5, 2), (12, 9), (40, 3)])
def test_blocks_that_share_keys(bfv, ctx, dim, seqs, group):
    """Eight, four, two blocks and one for a key head, with dims that fill the padded rows and dims that do not: every block
    is there until the others have read its part.  Many calls in a row give the same bits."""
    heads, length = 8, 300
    lens = [length - 7 * s % 290 for s in range(seqs)]
    kv, cache, table, lengths, held = filled(bfv, ctx, lens, heads, dim)
    q = randn(torch.Generator().manual_seed(5), seqs, heads * group, dim)
    first = kv.decode(q.cuda(), table, lengths)
    rest = [kv.decode(q.cuda(), table, lengths) for _ in range(20)]
    assert ctx.check() == 0
    assert all(torch.equal(first, x) for x in rest)
    for s in range(0, seqs, 4):
        want, bound = R.attention(q[s:s + 1], *held[s], lens[s], 0, 0, dim ** -0.5, two_terms=True)
        check(first[s:s + 1], want, bound)


@pytest.mark.parametrize("dim", [24, 72, 128])
def test_blocks_that_share_keys_in_parts(bfv, ctx, dim):
    """One sequence long enough for several groups of eight blocks, whose parts another kernel joins."""
    kv, cache, table, lengths, held = filled(bfv, ctx, [9000], 1, dim, page=64)
    q = randn(torch.Generator().manual_seed(5), 1, 12, dim)
    first = kv.decode(q.cuda(), table, lengths)
    assert all(torch.equal(first, kv.decode(q.cuda(), table, lengths)) for _ in range(20))
    assert ctx.check() == 0
    want, bound = R.attention(q, *held[0], 9000, 0, 0, dim ** -0.5, two_terms=True)
    check(first, want, bound)


@pytest.mark.parametrize("tokens,seqs", [(9, 2), (600, 2), (600, 40)])
def test_starts_that_leave_tokens_out_are_recorded(bfv, ctx, tokens, seqs):
    """Tokens before the first sequence's or after the last one's: recorded by prompt as by append, whichever kernel it is;
    the rows of the others are what they are anyway."""
    heads, dim = 8, 128
    kv, cache, table, lengths, held = filled(bfv, ctx, [tokens] * 2 + [16] * (seqs - 2), heads, dim)
    q = randn(torch.Generator().manual_seed(5), tokens, 2 * heads, dim).cuda()
    k = q[:, :heads].contiguous()
    rest = [0] * (seqs - 2)
    good = ints([0, tokens - 3, tokens] + [tokens for _ in rest])
    want = kv.prompt(q, good, table, lengths)
    assert ctx.check() == 0
    some_left_out = ((0, tokens - 3, tokens - 1), (2, tokens - 3, tokens), (0, 0, 0), (0, tokens - 3, tokens - 3))
    for a, b, c in some_left_out:
        starts = ints([a, b, c] + [c for _ in rest])
        out = torch.zeros_like(q)
        kv.prompt(q, starts, table, lengths, out=out)
        with pytest.raises(bfv.BfvGpuError, match="E_KV_TABLE"):
            ctx.check()
        assert (out[:a] == 0).all() and (out[c:] == 0).all()
        if b == tokens - 3:
            assert torch.equal(out[a:b], want[a:b])
    for a, b, c in some_left_out:  # (these change the cache)
        kv.append(k, k, ints([a, b, c] + [c for _ in rest]), table, lengths)
        with pytest.raises(bfv.BfvGpuError, match="E_KV_TABLE"):
            ctx.check()
    assert ctx.check() == 0


def test_tensors_let_go_during_a_call_on_another_stream(bfv, ctx):
    """What a call on a named stream reads and writes is not given out again before its work is done."""
    gen = torch.Generator().manual_seed(5)
    lens = [700, 90, 33]
    kv, cache, table, lengths, held = filled(bfv, ctx, lens, 2, 64)
    q, k, v = (randn(gen, 3, h, 64).cuda() for h in (4, 2, 2))
    starts = ints([0, 1, 2, 3])
    before = cache.k.clone(), cache.v.clone()
    kv.append(k, v, starts, table, lengths)
    want = kv.decode(q, table, lengths)
    want_p = kv.prompt(q, starts, table, lengths)
    cache.k.copy_(before[0])
    cache.v.copy_(before[1])
    page = int(table[1, 0])
    src, dst = ints([page]), ints([int(cache.spare[0])])
    fresh, rows = ints([int(cache.spare[1])]), ints([0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    handle = side.cuda_stream
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)
    out = torch.empty_like(q)
    given = [[x.clone() for x in args] for args in (
        (k, v, starts, table, lengths), (q, table, lengths, out), (q, starts, table, lengths, out), (src, dst, table),
        (rows, ints([2]), fresh, table, lengths))]
    torch.cuda.current_stream().synchronize()  # (the copies are there; the other stream still sleeps)
    used = {x.data_ptr() for args in given for x in args}
    kv.append(*given[0], stream=handle)
    kv.decode(*given[1][:3], out=given[1][3], stream=handle)
    kv.prompt(*given[2][:4], out=given[2][4], stream=handle)
    kv.move(*given[3], stream=handle)
    kv.fork(*given[4], stream=handle)
    got, got_p = given[1][3], given[2][4]
    shapes = [(x.shape, x.dtype) for args in given for x in args for _ in range(2)]
    got_at = {got.data_ptr(), got_p.data_ptr()}
    del given
    others = [torch.zeros(shape, dtype=dtype, device="cuda") for shape, dtype in shapes]
    assert not side.query()
    assert not used & {x.data_ptr() for x in others} and not got_at & {x.data_ptr() for x in others}
    side.synchronize()
    assert ctx.check() == 0
    assert torch.equal(got, want) and torch.equal(got_p, want_p)


def test_pages_let_go_during_a_call_on_another_stream(bfv, ctx):
    gen = torch.Generator().manual_seed(5)
    kv, cache, table, lengths, held = filled(bfv, ctx, [50])
    k = randn(gen, 1, 2, 64).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)
    kv.append(k, k, None, table, lengths, stream=side.cuda_stream)
    pages = {cache.k.data_ptr(), cache.v.data_ptr()}
    shape = cache.k.shape
    del kv, cache
    others = [torch.empty(shape, dtype=BF, device="cuda") for _ in range(4)]
    assert not side.query()
    assert not pages & {x.data_ptr() for x in others}
    side.synchronize()
    assert ctx.check() == 0


def test_a_graph_of_calls_on_a_named_stream(bfv, ctx):
    """Captured with the capturing stream's handle, tensors let go after the capture, replayed."""
    kv, cache, table, lengths, held = filled(bfv, ctx, [700, 90, 33])
    q = randn(torch.Generator().manual_seed(5), 3, 4, 64).cuda()
    want = kv.decode(q, table, lengths)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = kv.decode(q, table, lengths, stream=side.cuda_stream)
        kv.decode(q * 2, table, lengths, stream=side.cuda_stream)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del graph
    assert ctx.check() == 0


@pytest.mark.parametrize("scale", [1e-37, 1e-39, 2e-45])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 64)])
def test_scales_below_the_normal_range(bfv, ctx, scale, dim, page):
    """Keys that a row does not see stay out of it for the smallest scales too, in both kernels."""
    from test_gpu_kv import run_attention
    for kind, lens in (("prompt", [(600, 600), (300, 40)]), ("prompt", [(60, 9)]), ("decode", [(600, 1), (9, 1)])):
        run_attention(bfv, ctx, kind, BF, lens, 4, 2, dim, page, scale=scale)
        run_attention(bfv, ctx, kind, BF, lens, 4, 2, dim, page, 50, 3, scale=scale)


@pytest.mark.parametrize("stride", [1001, 3, 0, 1 << 40])
def test_the_stride_of_a_single_element_is_not_used(bfv, ctx, stride):
    """One token, or one head: whatever the stride of that axis, as for the cache's own axes."""
    gen = torch.Generator().manual_seed(5)
    for heads, group, tokens, new in ((2, 2, 700, 1), (1, 1, 90, 90), (1, 1, 1500, 1500)):
        kv, cache, table, lengths, held = filled(bfv, ctx, [tokens], heads, 64)
        h = heads * group
        dense = randn(gen, new, h, 64).cuda()
        odd = dense.as_strided(dense.shape, (stride if new == 1 else h * 64, stride if h == 1 else 64, 1))
        starts = ints([0, new])
        assert torch.equal(kv.prompt(odd, starts, table, lengths), kv.prompt(dense, starts, table, lengths))
        if new == 1:
            assert torch.equal(kv.decode(odd, table, lengths), kv.decode(dense, table, lengths))
        for dtype in (BF, torch.float32):
            k = dense[:, :heads].to(dtype)
            odd_k = k.as_strided(k.shape, (stride if new == 1 else heads * 64, stride if heads == 1 else 64, 1))
            kv.append(odd_k, odd_k, starts, table, lengths)
            p, r = cache.where(0)
            assert torch.equal(cache.k[0, p[-new:].cuda(), :, r[-new:].cuda()], dense[:, :heads])
            cache.put(0, *held[0])
    assert ctx.check() == 0
