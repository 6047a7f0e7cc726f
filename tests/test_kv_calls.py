"""What PagedKv hands to its calls, without a GPU."""
from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")

ARGUMENT = 1


class Pages:
    """What PagedKv asks of a tensor of pages."""

    shape, dtype = (1, 4, 2, 16, 64), torch.bfloat16
    device = types.SimpleNamespace(type="cuda", index=-1)

    def dim(self):
        return len(self.shape)

    def stride(self, axis=None):
        strides = 8192, 2048, 1024, 64, 1
        return strides if axis is None else strides[axis]

    def data_ptr(self):
        return 0x10000


def test_a_closed_context_is_not_used(bfv, monkeypatch):
    """Every call hands over the context as it is then: none once it is closed, which the C ABI refuses."""
    from bfvgpu import kvcache
    given = []

    class Calls:
        def open(self, *a):
            return "cache"

        def __getattr__(self, name):
            def call(cache, ctx, *rest):
                given.append(ctx)
                return 0 if ctx else bfv.lib().bfvgpu_kv_append_device(None, bfv._lib.KvDesc(
                    0x10000, 0x10000, 0, 1, 4, 2, 16, 64, 8192, 2048, 1024, 64), 0, None, None, 0, 0, 0, 0, None, None, 0,
                    None, 0, None)
            return call

    monkeypatch.setattr(kvcache, "_module", Calls())
    ctx = bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=-1)
    kv = bfv.PagedKv(ctx, Pages(), Pages())
    calls = [lambda: kv.append(1, 2, 3, 4, 5), lambda: kv.fork(1, 2, 3, 4, 5), lambda: kv.move(1, 2),
             lambda: kv.decode(1, 2, 3), lambda: kv.prompt(1, 2, 3, 4)]
    for call in calls:
        call()
    assert given == [ctx.handle.value] * len(calls)
    ctx.close()
    given.clear()
    for call in calls:
        with pytest.raises(bfv.BfvGpuInvalidArgument, match="E_BFVGPU_ARGUMENT") as refused:
            call()
        assert refused.value.code == ARGUMENT
    assert given == [None] * len(calls)


def test_the_library_builds_without_torch(bfv, monkeypatch, tmp_path):
    """The C library needs no torch: without it, only the module of the calls on torch tensors is left out, and what is
    built is not called stale for the lack of it."""
    import importlib.util

    import build as B
    ran = []
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libbfvgpu.so"))
    monkeypatch.setattr(B, "CALLS", str(tmp_path / "bfvgpu_kv_calls.so"))
    monkeypatch.setattr(B, "PKG", str(tmp_path))
    (tmp_path / "lib").mkdir()

    def run(command, check):
        ran.append(command)
        open(command[command.index("-o") + 1], "w").close()

    monkeypatch.setattr(B.subprocess, "run", run)
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert B.stale()
    assert B.build() == B.LIB
    assert ran and not any(B.CALLS in c for c in ran)
    assert not B.stale()
    monkeypatch.setattr(importlib.util, "find_spec", find)
    assert B.stale()  # torch is there now, and the module is not
    B.build()
    assert any(B.CALLS in c for c in ran)
    assert not B.stale()


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38, 1e-50, -1e-39])
def test_scales_that_32_bits_do_not_hold_are_refused(bfv, scale):
    """The kernels work with scale log2(e): beyond 32 bits every score of 0 would be NaN."""
    import ctypes

    from bfvgpu._lib import KvDesc
    host = bfv.Context(4096, bfv.find_primes(4096, [36, 36, 37]), 2, 1, 65537, device=-1)
    cache = KvDesc(0x10000, 0x20000, 0, 1, 4, 2, 16, 64, 8192, 2048, 1024, 64)
    at = 0x30000
    L = bfv.lib()

    def status(scale):
        return (L.bfvgpu_kv_decode_device(host.handle, ctypes.byref(cache), 0, at, 256, 64, 4, at, 4, at, 2, 0, 0, scale, at, at,
                                          None),
                L.bfvgpu_kv_prompt_device(host.handle, ctypes.byref(cache), 0, at, 256, 64, 4, 9, at, at, 4, at, 2, 0, 0, scale,
                                          at, at, None))

    assert status(scale) == (ARGUMENT, ARGUMENT) and L.bfvgpu_last_error() == b"E_KV_SCALE"
    for good in (2.3e38, 1.0, 1e-39, 2e-45):
        assert status(good) == (10, 10) and L.bfvgpu_last_error() == b"E_BFVGPU_HOST_ONLY_CONTEXT"


def test_the_choice_of_the_prompt_kernel(bfv):
    """By sizes and strides; -1 and a message for sizes that the call refuses."""
    import ctypes

    from bfvgpu._lib import KvDesc
    L = bfv.lib()

    def kernel(tokens, seqs, keys, heads=8, group=2, dim=128, window=0, sinks=0, head_stride=None, token_stride=None, page=16):
        cache = KvDesc(0x10000, 0x20000, 0, 1, 4, heads, page, dim, 0, heads * page * dim, page * dim, dim)
        return L.bfvgpu_kv_prompt_kernel(ctypes.byref(cache), heads * group * dim if token_stride is None else token_stride,
                                         dim if head_stride is None else head_stride, heads * group, tokens, seqs,
                                         keys // page, window, sinks)

    rows, tiles = 0, 1
    assert [kernel(n, 1, 512) for n in (1, 16, 64, 128, 512)] == [rows, rows, rows, tiles, tiles]
    assert kernel(4 * 198, 4, 208, heads=4, group=8, window=14) == tiles
    assert kernel(64 * 16, 64, 5392, group=1, dim=64) == rows and kernel(64 * 17, 64, 5392, group=1, dim=64) == tiles
    assert kernel(128 * 4, 128, 3472, group=1) == rows and kernel(128 * 5, 128, 3472, group=1) == tiles
    for strides in (dict(head_stride=0), dict(token_stride=0), dict(head_stride=1 << 38), dict(token_stride=-8)):
        assert kernel(512, 1, 512, **strides) == rows  # broadcast, reversed, too far for the loads
    assert kernel(512, 1, 512, heads=1, group=1, dim=64, head_stride=0) == kernel(512, 1, 512, heads=1, group=1, dim=64)
    assert kernel(512, 1, 512, window=-1) == -1 and L.bfvgpu_last_error() == b"E_KV_WINDOW"
    assert kernel(512, 1, 512, dim=60) == -1 and L.bfvgpu_last_error() == b"E_KV_DIM"
    assert L.bfvgpu_kv_prompt_kernel(None, 8, 8, 1, 1, 1, 1, 0, 0) == -1
