"""Key-value cache in pages and the attention that reads it.

The protocol runs a decoder layer's linear calls; between the q/k/v call and the o call the party
that holds the decrypted projections (a client that computes the non-linear steps itself, or a
plaintext check of the protocol) needs a cache and its attention.  The reference has neither: its
attention is a two-party integer protocol.

* ``PagedKv``: the pages and the device calls on them (bfvgpu_kv_* of include/bfvgpu.h);
* ``KvCache``: the book-keeping of a set of sequences over them: pages handed out, shared by forks,
  freed and compacted on the host, in step with the device's table and lengths.

Torch provides device memory; the arithmetic is the library's kernels.  Calls run on torch's current
stream unless ``stream`` names another (a raw handle, 0 or None: the current one).
"""
from __future__ import annotations

import ctypes
import heapq

import numpy as np

from ._lib import BfvGpuError, KvDesc, check, lib
from .backend import Context

_LEGACY_STREAM = 1  # cudaStreamLegacy: the C ABI reads a null stream as the context's


def _dtypes():
    import torch
    return {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class PagedKv:
    """Pages k, v [layers][pages][heads][page_tokens][dim] (or without the layers axis), bfloat16 or
    float16 CUDA tensors of the same shape and strides, dim contiguous; the outer axes may lie in
    any order (pass a transposed view).  table [rows][width], lengths, starts, page and row lists:
    dense int32 CUDA tensors."""

    def __init__(self, ctx: Context, k, v):
        import torch
        self._torch = torch
        self._codes = _dtypes()
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
        self._desc = KvDesc(k.data_ptr(), v.data_ptr(), self._codes[k.dtype], self.layers, self.pages, self.heads,
                            self.page_tokens, self.dim, st[0], st[1], st[2], st[3])
        # what every call needs, looked up once: these calls last microseconds
        L = lib()
        self._ref, self._index, self._int32 = ctypes.byref(self._desc), ctx.device, torch.int32
        self._append, self._fork, self._move = L.bfvgpu_kv_append_device, L.bfvgpu_kv_fork_device, L.bfvgpu_kv_move_device
        self._decode, self._prompt = L.bfvgpu_kv_decode_device, L.bfvgpu_kv_prompt_device
        self._scale = self.dim ** -0.5
        self._current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        self._scratch_words = {}  # by the sizes of a call

    # ---- helpers ----
    def _stream(self, stream) -> int:
        return int(stream) if stream else self._current_stream(self._index) or _LEGACY_STREAM

    def _table(self, table):
        """(address, rows, width)"""
        if table.dtype is not self._int32 or table.get_device() != self._index or table.dim() != 2 or (
                not table.is_contiguous()):
            raise ValueError("E_KV_SHAPE: the table is a dense int32 tensor [rows][width] on the cache's device")
        rows, width = table.shape
        return table.data_ptr(), rows, width

    def _ints(self, t, name: str, count: int) -> int:
        if t.dtype is not self._int32 or t.get_device() != self._index or t.dim() != 1 or t.shape[0] != count or (
                not t.is_contiguous()):
            raise ValueError(f"E_KV_SHAPE: {name} is a dense int32 tensor [{count}] on the cache's device")
        return t.data_ptr()

    def _rows(self, t, name: str):
        """(tokens, heads, token stride, head stride)"""
        if t.dim() != 3 or t.get_device() != self._index:
            raise ValueError(f"E_KV_SHAPE: {name} is [tokens][heads][{self.dim}] on the cache's device")
        (tokens, heads, dim), (ts, hs, ds) = t.shape, t.stride()
        if dim != self.dim or ds != 1:
            raise ValueError(f"E_KV_SHAPE: {name} is [tokens][heads][{self.dim}], dim contiguous")
        return tokens, heads, ts, hs

    def _on(self, stream):
        """Allocations inside belong to the stream that the call runs on."""
        t = self._torch
        return t.cuda.stream(t.cuda.ExternalStream(int(stream), device=self.k.device))

    def _results(self, q, out, key, query, stream):
        """out, and the scratch of a call with these sizes."""
        t = self._torch
        words = self._scratch_words.get(key)
        if words is None:
            if len(self._scratch_words) >= 4096:
                self._scratch_words.clear()
            words = self._scratch_words[key] = int(query())
        if q.dtype is not self.k.dtype:
            raise ValueError("E_KV_DTYPE: q has the cache's type")
        if stream:
            with self._on(stream):
                return self._results(q, out, key, query, None)
        if out is None:
            out = t.empty_like(q, memory_format=t.contiguous_format)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.device != q.device or not out.is_contiguous():
            raise ValueError("E_KV_SHAPE: out is dense, of q's shape and type")
        return out, t.empty(words, dtype=t.int64, device=self.k.device) if words else None

    # ---- device calls ----
    def append(self, k_new, v_new, starts, table, lengths, layer: int = 0, stream: int | None = None) -> None:
        """New keys and values [tokens][heads][dim] (the cache's type, or float32 rounded to nearest)
        into the pages of their sequences: the last starts[s+1] - starts[s] of the lengths[s] tokens
        of sequence s (starts None: one each).  bfvgpu_kv_append_device."""
        tokens, heads, ts, hs = self._rows(k_new, "k_new")
        source = self._codes.get(k_new.dtype)
        if heads != self.heads or source not in (self._desc.dtype, 2):
            raise ValueError("E_KV_SHAPE: k_new has the cache's heads, and its type or float32")
        if v_new.shape != k_new.shape or v_new.stride() != k_new.stride() or v_new.dtype is not k_new.dtype or (
                v_new.get_device() != self._index):
            raise ValueError("E_KV_SHAPE: k_new and v_new need one shape, type and layout")
        at, seqs, width = self._table(table)
        check(self._append(self.ctx.handle, self._ref, layer, k_new.data_ptr(), v_new.data_ptr(), source, ts, hs, tokens,
                           None if starts is None else self._ints(starts, "starts", seqs + 1), at, width,
                           self._ints(lengths, "lengths", seqs), seqs, self._stream(stream)), "kv_append_device")

    def fork(self, parents, children, fresh, table, lengths, stream: int | None = None) -> None:
        """Rows children[i] of the table continue rows parents[i]; a partly filled last page is copied
        to page fresh[i].  bfvgpu_kv_fork_device."""
        at, rows, width = self._table(table)
        n = parents.shape[0]
        check(self._fork(self.ctx.handle, self._ref, self._ints(parents, "parents", n), self._ints(children, "children", n),
                         self._ints(fresh, "fresh", n), n, at, rows, width, self._ints(lengths, "lengths", rows),
                         self._stream(stream)), "kv_fork_device")

    def move(self, src, dst, table=None, stream: int | None = None) -> None:
        """Pages src[i] (strictly increasing) to pages dst[i], all layers, and the table's entries
        with them.  bfvgpu_kv_move_device."""
        at, rows, width = (None, 0, 0) if table is None else self._table(table)
        n = src.shape[0]
        check(self._move(self.ctx.handle, self._ref, self._ints(src, "src", n), self._ints(dst, "dst", n), n, at, rows, width,
                         self._stream(stream)), "kv_move_device")

    def decode(self, q, table, lengths, layer: int = 0, window: int = 0, sinks: int = 0, scale: float | None = None,
               out=None, stream: int | None = None):
        """Attention of the newest token of every sequence: q [seqs][q_heads][dim] of the cache's type
        -> out [seqs][q_heads][dim].  window 0: all keys; else the last `window` keys and the first
        `sinks`.  scale None: dim ** -0.5.  bfvgpu_kv_decode_device."""
        tokens, h, ts, hs = self._rows(q, "q")
        at, seqs, width = self._table(table)
        if tokens != seqs:
            raise ValueError("E_KV_SHAPE: one query per row of the table")
        out, scratch = self._results(q, out, (h, seqs, width, window, sinks), lambda: lib().bfvgpu_kv_decode_scratch_words(
            self.ctx.handle, self._ref, h, seqs, width, window, sinks), stream)
        check(self._decode(self.ctx.handle, self._ref, layer, q.data_ptr(), ts, hs, h, at, width,
                           self._ints(lengths, "lengths", seqs), seqs, window, sinks, self._scale if scale is None else scale,
                           None if scratch is None else scratch.data_ptr(), out.data_ptr(), self._stream(stream)),
              "kv_decode_device")
        return out

    def prompt(self, q, starts, table, lengths, layer: int = 0, window: int = 0, sinks: int = 0,
               scale: float | None = None, out=None, stream: int | None = None):
        """The same for the new tokens of every sequence: q [tokens][q_heads][dim], sequence s having
        rows starts[s] .. starts[s+1] - 1, its last tokens.  bfvgpu_kv_prompt_device."""
        tokens, h, ts, hs = self._rows(q, "q")
        at, seqs, width = self._table(table)
        out, scratch = self._results(q, out, (h, tokens, seqs, width, window, sinks),
                                     lambda: lib().bfvgpu_kv_prompt_scratch_words(
                                         self.ctx.handle, self._ref, h, tokens, seqs, width, window, sinks), stream)
        check(self._prompt(self.ctx.handle, self._ref, layer, q.data_ptr(), ts, hs, h, tokens,
                           self._ints(starts, "starts", seqs + 1), at, width, self._ints(lengths, "lengths", seqs), seqs,
                           window, sinks, self._scale if scale is None else scale, None if scratch is None else scratch.data_ptr(),
                           out.data_ptr(), self._stream(stream)), "kv_prompt_device")
        return out


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
        """The attention of the step's tokens, after append: q [tokens][q_heads][dim]."""
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
