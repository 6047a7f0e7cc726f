"""Key-value cache in pages and the attention that reads it.

The protocol runs a decoder layer's linear calls; between the q/k/v call and the o call the party
that holds the decrypted projections (a client that computes the non-linear steps itself, or a
plaintext check of the protocol) needs a cache and its attention (head norms and positions, where
the model has them, are its own).  The reference has neither: its
attention is a two-party integer protocol.

* ``PagedKv``: the pages and the device calls on them (bfvgpu_kv_* of include/bfvgpu.h);
* ``KvCache``: the book-keeping of a set of sequences over them: pages handed out, shared by forks,
  freed and compacted on the host, in step with the device's table and lengths.

Torch provides device memory; the arithmetic is the library's kernels.  Calls run on torch's current
stream unless ``stream`` names another (a raw handle, 0 or None: the current one).  On a named stream the
caller orders the call after what it reads; its tensors may be let go at once, as after
``Tensor.record_stream``, and what it returns belongs to that stream.
"""
from __future__ import annotations

import ctypes
import heapq
import importlib.util
import os

import numpy as np

from ._lib import LIB_PATH, BfvGpuError, BfvGpuUnavailable, KvDesc, check, lib
from .backend import Context

_module = None


def _calls():
    """The module of the calls on torch tensors (csrc/kv_torch.cpp), built beside the library."""
    global _module
    if _module is None:
        import torch  # noqa: F401  (its libraries are the module's)
        lib()
        path = os.path.join(os.path.dirname(LIB_PATH), "bfvgpu_kv_calls.so")
        if not os.path.exists(path):
            raise BfvGpuUnavailable(f"{path} is not built (python privacy-rag_b200/build.py)")
        spec = importlib.util.spec_from_file_location("bfvgpu_kv_calls", path)
        _module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_module)
    return _module


class PagedKv:
    """Pages k, v [layers][pages][heads][page_tokens][dim] (or without the layers axis), bfloat16 or
    float16 CUDA tensors of the same shape and strides, dim contiguous; the outer axes may lie in
    any order (pass a transposed view).  table [rows][width], lengths, starts, page and row lists:
    dense int32 CUDA tensors.  For serving: no gradient passes through a call, what it returns or
    writes is cut off from its arguments' graph."""

    def __init__(self, ctx: Context, k, v):
        import torch
        if k.dim() == 4:
            k, v = k.unsqueeze(0), v.unsqueeze(0)
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.stride(4) != 1:
            raise ValueError("E_KV_SHAPE: k and v need one shape, type and layout, dim contiguous")
        if k.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("E_KV_DTYPE")
        if k.device != v.device or k.device.type != "cuda" or k.device.index != ctx.device:
            raise ValueError("E_KV_DEVICE: pages live on the context's device")
        self.ctx, self.k, self.v = ctx, k, v
        self.layers, self.pages, self.heads, self.page_tokens, self.dim = (int(x) for x in k.shape)
        st = k.stride()
        desc = KvDesc(k.data_ptr(), v.data_ptr(), 0 if k.dtype == torch.bfloat16 else 1, self.layers, self.pages, self.heads,
                      self.page_tokens, self.dim, st[0], st[1], st[2], st[3])
        self._calls, self._desc = _calls(), desc
        self._cache = self._calls.open(ctypes.addressof(desc), ctx.device, k, v)

    @property
    def _handle(self) -> int | None:
        """The context as it is now: None once it is closed, which the calls refuse."""
        h = self.ctx.handle
        return h.value if h is not None else None

    # ---- device calls ----
    def append(self, k_new, v_new, starts, table, lengths, layer: int = 0, stream: int | None = None) -> None:
        """New keys and values [tokens][heads][dim] (the cache's type, or float32 rounded to nearest)
        into the pages of their sequences: the last starts[s+1] - starts[s] of the lengths[s] tokens
        of sequence s (starts None: one each).  bfvgpu_kv_append_device."""
        check(self._calls.append(self._cache, self._handle, k_new, v_new, starts, table, lengths, layer, stream),
              "kv_append_device")

    def fork(self, parents, children, fresh, table, lengths, stream: int | None = None) -> None:
        """Rows children[i] of the table continue rows parents[i]; a partly filled last page is copied
        to page fresh[i].  bfvgpu_kv_fork_device."""
        check(self._calls.fork(self._cache, self._handle, parents, children, fresh, table, lengths, stream), "kv_fork_device")

    def move(self, src, dst, table=None, stream: int | None = None) -> None:
        """Pages src[i] (strictly increasing) to pages dst[i], all layers, and the table's entries
        with them.  bfvgpu_kv_move_device."""
        check(self._calls.move(self._cache, self._handle, src, dst, table, stream), "kv_move_device")

    def decode(self, q, table, lengths, layer: int = 0, window: int = 0, sinks: int = 0, scale: float | None = None,
               out=None, stream: int | None = None):
        """Attention of the newest token of every sequence: q [seqs][q_heads][dim] of the cache's type
        -> out [seqs][q_heads][dim].  window 0: all keys; else the last `window` keys and the first
        `sinks`.  scale None: dim ** -0.5.  bfvgpu_kv_decode_device."""
        r = self._calls.decode(self._cache, self._handle, q, table, lengths, layer, window, sinks, scale, out, stream)
        if type(r) is int:
            check(r, "kv_decode_device")
        return r

    def prompt(self, q, starts, table, lengths, layer: int = 0, window: int = 0, sinks: int = 0,
               scale: float | None = None, out=None, stream: int | None = None):
        """The same for the new tokens of every sequence: q [tokens][q_heads][dim], sequence s having
        rows starts[s] .. starts[s+1] - 1, its last tokens; every row belongs to a sequence.  The values of a
        token that some rows of a block of 256 see have to be finite for the block's others too (0 x NaN);
        what none of them sees may hold anything.  bfvgpu_kv_prompt_device."""
        r = self._calls.prompt(self._cache, self._handle, q, starts, table, lengths, layer, window, sinks, scale, out, stream)
        if type(r) is int:
            check(r, "kv_prompt_device")
        return r

    def prompt_kernel(self, q, table, window: int = 0, sinks: int = 0) -> str:
        """Which kernel ``prompt`` takes, by sizes and strides alone: "rows", as every ``decode``, whose weights
        keep the remainder of their rounding to 16 bits, or "tiles", the tensor-core kernel, whose weights do
        not.  bfvgpu_kv_prompt_kernel."""
        kernel = lib().bfvgpu_kv_prompt_kernel(ctypes.byref(self._desc), q.stride(0), q.stride(1), q.shape[1], q.shape[0],
                                               table.shape[0], table.shape[1], window, sinks)
        if kernel < 0:
            raise ValueError(lib().bfvgpu_last_error().decode())
        return ("rows", "tiles")[kernel]


class PageBook:
    """Host book-keeping of the pages: which page holds which tokens of which sequence.  Full pages
    may be shared (a fork copies a partly filled last page, so tokens are only ever written to a page
    of one sequence).  Pages are handed out lowest number first.  A request that does not fit changes
    nothing and raises BfvGpuError (BFVGPU_E_ALLOC, E_KV_PAGES)."""

    def __init__(self, pages: int, page_tokens: int, sequences: int, width: int):
        if pages < 1 or page_tokens < 1 or sequences < 1 or width < 1:
            raise ValueError("E_KV_SHAPE")
        self.page_tokens, self.width = page_tokens, width
        self.table = np.full((sequences, width), -1, dtype=np.int32)
        self.lengths = np.zeros(sequences, dtype=np.int32)
        self.refs = np.zeros(pages, dtype=np.int32)
        self.active = np.zeros(sequences, dtype=bool)
        self._free = list(range(pages))  # a heap

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _row(self, row: int) -> int:
        if not 0 <= row < len(self.lengths) or not self.active[row]:
            raise ValueError(f"E_KV_ROW: {row}")
        return row

    def _need(self, pages: int) -> None:
        if pages > len(self._free):
            raise BfvGpuError(14, f"E_KV_PAGES: {pages} wanted, {len(self._free)} free", "KvCache")

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self.refs[p] = 1
        return p

    def _drop(self, page: int) -> None:
        self.refs[page] -= 1
        if self.refs[page] == 0:
            heapq.heappush(self._free, int(page))

    def _rows_free(self, count: int) -> list[int]:
        rows = np.flatnonzero(~self.active)[:count]
        if len(rows) < count:
            raise BfvGpuError(14, f"E_KV_ROWS: {count} wanted, {len(rows)} free", "KvCache")
        return [int(r) for r in rows]

    def open(self) -> int:
        """A new empty sequence; its row."""
        row = self._rows_free(1)[0]
        self.active[row] = True
        return row

    def extend(self, counts: dict[int, int]) -> None:
        """counts[row] more tokens for each row."""
        grow = {}
        for row, n in counts.items():
            self._row(row)
            have, want = int(self.lengths[row]), int(self.lengths[row]) + int(n)
            if n < 0 or want > self.width * self.page_tokens:
                raise ValueError(f"E_KV_LENGTH: row {row}: {have} + {n} tokens")
            grow[row] = range(-(-have // self.page_tokens), -(-want // self.page_tokens))
        self._need(sum(len(g) for g in grow.values()))
        for row, slots in grow.items():
            for slot in slots:
                self.table[row, slot] = self._take()
            self.lengths[row] += counts[row]

    def fork(self, row: int, count: int) -> tuple[list[int], list[int]]:
        """count new sequences that continue `row`; (their rows, the page of each that takes a copy
        of the partly filled last page, -1 where there is none)."""
        self._row(row)
        if count < 0:
            raise ValueError("E_KV_SHAPE")
        children = self._rows_free(count)
        n = int(self.lengths[row])
        last, part = n // self.page_tokens, n % self.page_tokens != 0
        self._need(count if part else 0)
        fresh = []
        for c in children:
            self.active[c] = True
            self.lengths[c] = n
            self.table[c] = self.table[row]
            if part:
                self.table[c, last] = self._take()
            for slot, page in enumerate(self.table[c]):
                if page >= 0 and not (part and slot == last):
                    self.refs[page] += 1
            fresh.append(int(self.table[c, last]) if part else -1)
        return children, fresh

    def free(self, row: int) -> None:
        """Ends a sequence."""
        self._row(row)
        for page in self.table[row][self.table[row] >= 0]:
            self._drop(page)
        self.table[row] = -1
        self.lengths[row] = 0
        self.active[row] = False

    def trim(self, window: int, sinks: int) -> int:
        """Gives up the pages that no later query with this window sees; how many entries."""
        if window < 1 or sinks < 0:
            raise ValueError("E_KV_WINDOW")
        gone = 0
        for row in np.flatnonzero(self.active):
            # the next query stands at p = length and sees j > p - window and j < sinks
            last = (int(self.lengths[row]) - window + 1) // self.page_tokens
            for slot in range(-(-sinks // self.page_tokens), max(0, last)):
                if self.table[row, slot] >= 0:
                    self._drop(self.table[row, slot])
                    self.table[row, slot] = -1
                    gone += 1
        return gone

    def compact(self) -> tuple[list[int], list[int]]:
        """Moves the pages in use to the lowest numbers: (src rising, dst rising); the table follows."""
        used = np.flatnonzero(self.refs > 0)
        holes = np.flatnonzero(self.refs[:len(used)] == 0)
        src = used[len(used) - len(holes):]
        to = np.arange(len(self.refs), dtype=np.int32)
        to[src] = holes
        self.table = np.where(self.table >= 0, to[np.maximum(self.table, 0)], -1).astype(np.int32)
        self.refs[holes] = self.refs[src]
        self.refs[src] = 0
        self._free = [int(p) for p in np.flatnonzero(self.refs == 0)]  # sorted, so a heap
        return [int(p) for p in src], [int(p) for p in holes]


class KvCache:
    """Sequences over one PagedKv: book-keeping on the host, table and lengths on the device in step.

    Every call covers all rows of the table (a row without a sequence, or without new tokens in this
    step, takes part with none), so the device side of a step has fixed shapes.  One step:
    ``extend`` the rows that get tokens, then per layer ``append`` their keys and values and
    ``attend``, with the tokens of the rows in row order."""

    def __init__(self, ctx: Context, pages: int, heads: int, dim: int, layers: int = 1, page_tokens: int = 16,
                 sequences: int = 64, tokens: int = 4096, dtype=None):
        """pages over all sequences; tokens: the longest sequence."""
        import torch
        self._torch, self.ctx = torch, ctx
        dev = torch.device("cuda", ctx.device)
        self.book = PageBook(pages, page_tokens, sequences, -(-tokens // page_tokens))
        # zeros: values of pages that nothing was written to yet may be copied by a fork
        shape = (layers, pages, heads, page_tokens, dim)
        dtype = dtype or torch.bfloat16
        self.kv = PagedKv(ctx, torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev))
        self.table = torch.full(self.book.table.shape, -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        self.starts = torch.zeros(sequences + 1, dtype=torch.int32, device=dev)
        self._each = 0  # 1: the step gives every row one token

    def _ints(self, values):
        return self._torch.tensor(values, dtype=self._torch.int32).pin_memory().to(self.table.device, non_blocking=True)

    def _push(self) -> None:
        """The host's table and lengths to the device, in the order of the current stream."""
        self.table.copy_(self._torch.from_numpy(self.book.table.copy()).pin_memory(), non_blocking=True)
        self.lengths.copy_(self._torch.from_numpy(self.book.lengths.copy()).pin_memory(), non_blocking=True)

    def open(self) -> int:
        return self.book.open()

    def extend(self, counts: dict[int, int]) -> None:
        """Begins a step: counts[row] new tokens for each row."""
        self.book.extend(counts)
        new = np.zeros(len(self.book.lengths), dtype=np.int64)
        for row, n in counts.items():
            new[row] = n
        self._each = int((new == 1).all())
        self.starts.copy_(self._ints(np.concatenate([[0], np.cumsum(new)]).tolist()), non_blocking=True)
        self._push()

    def append(self, k_new, v_new, layer: int = 0) -> None:
        """The step's keys and values [tokens][heads][dim] of one layer."""
        self.kv.append(k_new, v_new, self.starts, self.table, self.lengths, layer=layer)

    def attend(self, q, layer: int = 0, window: int = 0, sinks: int = 0, scale: float | None = None, out=None):
        """The attention of the step's tokens, after append: q [tokens][q_heads][dim].  A ``decode`` where
        every row of the table gets one token, else a ``prompt`` of all rows, whose kernel goes by their number
        and the table's width (``PagedKv.prompt_kernel``)."""
        if self._each:
            return self.kv.decode(q, self.table, self.lengths, layer, window, sinks, scale, out)
        return self.kv.prompt(q, self.starts, self.table, self.lengths, layer, window, sinks, scale, out)

    def fork(self, row: int, count: int = 1) -> list[int]:
        """count sequences that continue `row`, sharing its full pages."""
        children, fresh = self.book.fork(row, count)
        if children:
            self.kv.fork(self._ints([row] * count), self._ints(children), self._ints(fresh), self.table, self.lengths)
        return children

    def free(self, row: int) -> None:
        self.book.free(row)
        self._push()

    def trim(self, window: int, sinks: int = 0) -> int:
        """Frees the pages that no later query with this window and these first tokens sees."""
        gone = self.book.trim(window, sinks)
        if gone:
            self._push()
        return gone

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers; how many moved."""
        src, dst = self.book.compact()
        if src:
            self.kv.move(self._ints(src), self._ints(dst), self.table)
        return len(src)
