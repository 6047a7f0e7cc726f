"""Rotary positions without a GPU: frequencies, their fractions of a turn, refusals."""
from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import pytest

ARGUMENT, SHAPE = 1, 3


@pytest.fixture
def host(bfv):
    return bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=-1)


def test_frequencies(bfv):
    from bfvgpu.rotary import frequencies
    w, scale = frequencies(128, 1e6)
    assert scale == 1.0 and w[0] == 1.0 and len(w) == 64 and math.isclose(w[-1], 1e6 ** (-126 / 128))
    assert frequencies(128, 1e6, "linear", 4.0)[0] == [x / 4 for x in w]
    ntk = frequencies(128, 1e6, "ntk", 4.0)[0]
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], w[-1] / 4)
    yarn, scale = frequencies(128, 1e6, "yarn", 4.0, trained=4096)
    assert scale == 0.1 * math.log(4) + 1
    turns = [4096 * x / (2 * math.pi) for x in w]
    assert all(a == b for a, b, t in zip(yarn, w, turns) if t > 40) and any(t > 40 for t in turns)
    assert all(math.isclose(a, b / 4) for a, b, t in zip(yarn, w, turns) if t < 0.8) and any(t < 0.8 for t in turns)
    assert all(b / 4 <= a * (1 + 1e-12) and a <= b for a, b in zip(yarn, w))
    assert all(a > b for a, b in zip(yarn, yarn[1:]))
    for bad in (dict(dims=7), dict(base=1.0), dict(base=math.inf), dict(factor=0.5), dict(factor=math.nan), dict(scaling="more"),
                dict(dims=2, scaling="ntk"), dict(scaling="yarn", turns=(32.0, 1.0)), dict(scaling="yarn", trained=0)):
        with pytest.raises(ValueError, match="E_ROTARY"):
            frequencies(**{**dict(dims=64), **bad})


def test_fractions_of_a_turn(bfv, host):
    """turns[i] / 2^64 is the frequency modulo a turn, to 2^-63."""
    pi = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)
    radians = [1.0, 1e-6, 0.0, -0.25, 2 * math.pi, 100.0, 3.0e5, 1e-30]
    r = bfv.Rotary(host, 16, radians=radians, scale=0.5)
    assert r.scale == 0.5 and r._desc.scale == 0.5 and r._desc.dims == 16 and r._desc.layout == 0
    for x, got in zip(radians, r._desc.turns):
        share = Fraction(x) / (2 * pi)
        off = (Fraction(got, 2 ** 64) - share) % 1
        # a division in extended precision: half a step of the quotient, 2^-64 of it
        assert min(off, 1 - off) <= Fraction(1, 2 ** 64) + abs(share) / 2 ** 63
    assert list(r._desc.turns)[8:] == [0] * 56


def test_rotary_refusals(bfv, host):
    for bad in (dict(dims=6), dict(dims=0), dict(dims=132), dict(layout="other"), dict(scaling="more"), dict(radians=[1.0]),
                dict(radians=[1.0] * 7 + [math.nan]), dict(radians=[1.0] * 7 + [math.inf]), dict(scale=math.inf),
                dict(scale=1e39)):
        with pytest.raises(ValueError, match="E_ROTARY"):
            bfv.Rotary(host, **{**dict(dims=16), **bad})


def test_calls_refuse(bfv, host):
    """Arguments are checked before the device is looked for."""
    from bfvgpu._lib import KvDesc, RotaryDesc
    L, at = bfv.lib(), 0x30000
    good = bfv.Rotary(host, 64)._desc

    def rotary(**kw):
        r = RotaryDesc()
        ctypes.memmove(ctypes.byref(r), ctypes.byref(good), ctypes.sizeof(r))
        for k, v in kw.items():
            setattr(r, k, v)
        return r

    def apply(r=good, dtype=0, dim=64, tokens=3, heads=2, norm=None, eps=1e-6, inverse=0, x=at):
        rc = L.bfvgpu_rotary_device(host.handle, ctypes.byref(r) if r else None, x, dtype, 128, 64, tokens, heads, dim, at, norm,
                                    eps, inverse, at, 128, 64, None)
        return rc, L.bfvgpu_last_error()

    here = (10, b"E_BFVGPU_HOST_ONLY_CONTEXT")
    assert apply() == here and apply(norm=at) == here and apply(inverse=1) == here and apply(dtype=2) == here
    assert apply(r=None) == (ARGUMENT, b"E_ROTARY_ARGUMENT")
    assert apply(r=rotary(layout=2)) == (ARGUMENT, b"E_ROTARY_LAYOUT")
    assert apply(r=rotary(scale=math.nan)) == (ARGUMENT, b"E_ROTARY_SCALE")
    for dims in (0, 2, 62, 68, 132, -4):
        assert apply(r=rotary(dims=dims)) == (SHAPE, b"E_ROTARY_DIMS")
    for dim in (0, 60, 136):
        assert apply(dim=dim) == (SHAPE, b"E_ROTARY_DIM")
    assert apply(dtype=3) == (ARGUMENT, b"E_ROTARY_DTYPE")
    assert apply(norm=at, inverse=1) == (ARGUMENT, b"E_ROTARY_NORM")
    assert apply(heads=1 << 16) == (SHAPE, b"E_ROTARY_SHAPE") and apply(tokens=1 << 31) == (SHAPE, b"E_ROTARY_SHAPE")
    for eps in (-1.0, math.nan, math.inf):
        assert apply(eps=eps) == (ARGUMENT, b"E_ROTARY_EPS")

    def append(cache=KvDesc(0x10000, 0x20000, 0, 1, 4, 2, 16, 64, 8192, 2048, 1024, 64), r=good, layer=0, source=2, q_heads=4,
               tokens=3, starts=at, width=4, seqs=2, eps=1e-6):
        rc = L.bfvgpu_kv_append_rotary_device(host.handle, ctypes.byref(cache), layer, ctypes.byref(r), at, at, source, 128, 64, at,
                                              256, 64, q_heads, None, None, eps, tokens, starts, at, width, at, seqs, at, None)
        return rc, L.bfvgpu_last_error()

    assert append() == here and append(q_heads=0) == here and append(source=0) == here
    assert append(source=1) == (ARGUMENT, b"E_KV_SOURCE_DTYPE")
    assert append(r=rotary(dims=68)) == (SHAPE, b"E_ROTARY_DIMS")
    assert append(layer=1) == (SHAPE, b"E_KV_LAYER") and append(layer=-1) == (SHAPE, b"E_KV_LAYER")
    assert append(starts=None) == (SHAPE, b"E_KV_STARTS")
    assert append(width=1 << 27) == (SHAPE, b"E_KV_WIDTH")
    assert append(q_heads=1 << 16) == (SHAPE, b"E_KV_SHAPE")
    assert append(eps=-1.0) == (ARGUMENT, b"E_ROTARY_EPS")
    assert L.bfvgpu_rotary_set(None, 8, 0, (ctypes.c_double * 4)(), 1.0) == ARGUMENT
    assert L.bfvgpu_rotary_set(ctypes.byref(RotaryDesc()), 8, 0, None, 1.0) == ARGUMENT
