"""The attention between two encrypted linear calls: a q/k/v call of the protocol (encryption, product,
masking, client phase on the GPU), its decoded words into RingAttention, forked answers and their next
tokens, against the attention of the same values in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import kv_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu

MASK = (1 << 59) - 1
Q_HEADS, KV_HEADS, DIM, INNER = 4, 2, 16, 64
FX, FW, F_OUT = 12, 8, 20


@pytest.fixture(scope="module")
def protocol(bfv, oracle):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from bfvgpu import engine
    hc, oc = bfv.Context.art002(0), oracle.art002()
    tb = oracle.TestBfv(oc, seed=77)
    rng = np.random.default_rng(5)
    q = np.array(hc.primes, dtype=np.int64).reshape(1, 1, -1, 1)

    def samples(g):
        u = rng.integers(-1, 2, size=(g, 1, 1, hc.n))
        e = rng.integers(-5, 6, size=(g, 2, 1, hc.n))
        return (np.concatenate([u, e], axis=1) % q).astype(np.uint64)

    client = engine.MatrixClient(hc, tb.pk, tb.sk_ntt, samples=samples)
    server = engine.MatrixServer(hc, tb.pk, masks=lambda g: rng.integers(0, 1 << 59, size=(g, hc.n), dtype=np.uint64),
                                 samples=samples)

    def call(x, w):
        """x [B][K], w [O][K] signed integers -> the call's decoded words [B][O], through both parties."""
        B, K = x.shape
        d, cap, blocks, tile = engine.plan(B, K, w.shape[0])
        words = x.astype(np.uint64) & np.uint64(MASK)
        wu = w.astype(np.uint64) & np.uint64(MASK)
        share = rng.integers(0, 1 << 59, size=words.shape, dtype=np.uint64)
        encrypted = client.encrypt_inputs(engine.pack_client_inputs(share, d, blocks, hc.n))
        result, tiles = server.run(encrypted, (words - share) & np.uint64(MASK), w.shape[0],
                                   lambda begin, actual, first, count: wu[first:first + count, begin:begin + actual],
                                   d, cap, B, tile)
        out = [[int(v) for v in row] for row in result]
        for t, u in zip(tiles, client.phases(tiles)):
            for i, (c0, c1) in enumerate(zip(t.c0_phase, u)):
                o, b = divmod(i, B)
                col = t.first_column + o
                out[b][col] = (out[b][col] + oracle.decode((c0 + c1) % oc.Q, oc.Q)) & MASK
        return np.array(out, dtype=np.int64)

    return hc, call


@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
def test_answers_of_one_prompt(bfv, protocol, window, sinks):
    hc, call = protocol
    rng = np.random.default_rng(9)
    width = (Q_HEADS + 2 * KV_HEADS) * DIM
    w = rng.integers(-60, 61, size=(width, INNER))
    att = bfv.RingAttention(hc, Q_HEADS, KV_HEADS, DIM, FX + FW, F_OUT, pages=12, page_tokens=16, sequences=3, tokens=64,
                            window=window, sinks=sinks)
    history = {}

    def step(counts):
        tokens = sum(counts.values())
        x = np.round(rng.standard_normal((tokens, INNER)) * 2 ** FX / 12).astype(np.int64)
        words = np.concatenate([call(x[i:i + 4], w) for i in range(0, tokens, 4)])
        assert np.array_equal(words, (x @ w.T) & MASK)  # the protocol's product is exact
        att.extend(counts)
        got = att.layer(torch.from_numpy(words).cuda()).cpu()
        value = torch.from_numpy(x @ w.T).double() * 2.0 ** -(FX + FW)
        rows = value.float().to(torch.bfloat16).unflatten(1, (Q_HEADS + 2 * KV_HEADS, DIM))
        at = 0
        for row in sorted(counts):
            n = counts[row]
            new = rows[at:at + n]
            k, v = history.get(row, (rows[:0, :KV_HEADS], rows[:0, :KV_HEADS]))
            k = torch.cat([k, new[:, Q_HEADS:Q_HEADS + KV_HEADS]])
            v = torch.cat([v, new[:, Q_HEADS + KV_HEADS:]])
            history[row] = k, v
            want, bound = R.attention(new[:, :Q_HEADS], k, v, len(k), window, sinks, DIM ** -0.5, two_terms=False)
            out = got[at:at + n]
            signed = torch.where(out >= 1 << 58, out - (1 << 59), out).double() * 2.0 ** -F_OUT
            error = (signed.unflatten(1, (Q_HEADS, DIM)) - want).abs()
            assert (error <= bound + 2.0 ** -(F_OUT + 1)).all()
            at += n
        assert hc.check() == 0

    doc = att.open()
    step({doc: 8})
    answers = att.fork(doc, 2)
    for a in answers:
        history[a] = history[doc]
    step({a: 1 for a in answers})
    att.free(doc)
    del history[doc]
    att.compact()
    step({answers[0]: 1, answers[1]: 3})
    step({a: 4 for a in answers})


def test_words_and_floats(bfv):
    from bfvgpu.attend import floats_to_words, words_to_floats
    values = torch.tensor([0, 1, -1, 5, (1 << 58) - 1, -(1 << 58), 3 << 20])
    words = values & MASK
    assert torch.equal(words_to_floats(torch, words, 0), values.float())
    assert torch.equal(words_to_floats(torch, words, 12), (values.double() / 4096).float())
    x = torch.tensor([0.0, 0.5, -0.5, 1.5, -1.5, 2.25, -7.0])
    assert floats_to_words(torch, x, 0).tolist() == [v & MASK for v in (0, 0, 0, 2, -2, 2, -7)]
    assert floats_to_words(torch, x, 2).tolist() == [v & MASK for v in (0, 2, -2, 6, -6, 9, -28)]
