"""Attention over a paged cache from its definition, in 64 bits on the CPU, with the bound that the
kernels' arithmetic allows.

For one query row with visible keys j: s_j = scale q.k_j, p_j = exp(s_j - max s), o = sum p_j v_j / sum p_j.
Let u be the unit roundoff of the 16-bit type (2^-8 for bfloat16, 2^-11 for float16), and
A = sum p_j |v_j| / sum p_j per output.  The error of one output is at most
  u |o|                        rounding of the result;
  up A                         rounding of each p_j before the product with v_j: up = u where the weights
                               enter the product in 16 bits; where they enter as two 16-bit terms their
                               sum is off by 2^-16 (bfloat16, u^2) or, for float16, u^2 p + 2^-25 (the
                               second term may be subnormal);
  2 e A                        relative error e of each p_j, in the numerator and in the sum: the score's
                               error in 32 bits, (dim + 4) 2^-24 scale max_j sum_d |q_d k_jd|, twice the
                               same from the shared maximum's own product (counted once more), 2^-21 for
                               the exponential, and (keys + 32) 2^-24 for sums of that many terms.
"""
from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def visible(pos, keys: int, window: int, sinks: int):
    """[rows][keys]: which keys a query at pos sees."""
    j = torch.arange(keys)[None, :]
    p = torch.as_tensor(pos)[:, None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    return seen


def rows(q, k, v, seen, scale: float, two_terms: bool):
    """q [n][d], k, v [keys][d], seen [n][keys] -> (o, bound) in 64 bits; rows that see nothing: 0, 0."""
    u = UNIT[q.dtype]
    q, k, v = q.double(), k.double(), v.double()
    any_seen = seen.any(0)  # what no row sees takes no part at all
    k, v = torch.where(any_seen[:, None], k, 0.0), torch.where(any_seen[:, None], v, 0.0)
    s = torch.where(seen, (q @ k.T) * scale, -math.inf)
    top = s.amax(1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(1, keepdim=True)
    norm = torch.where(total > 0, total, 1.0)
    o = (p @ v) / norm
    a = (p @ v.abs()) / norm
    size = torch.where(seen, (q.abs() @ k.abs().T) * scale, 0.0).amax(1, keepdim=True)
    e = 2 * (q.shape[1] + 4) * 2.0 ** -24 * size + 2.0 ** -21 + (k.shape[0] + 32) * 2.0 ** -24
    up = u * u + (2.0 ** -25 if u < 2.0 ** -9 else 0.0) if two_terms else u
    # a float16 weight below 2^-14 is rounded to a multiple of 2^-24, whatever its size
    tiny = 0.0 if two_terms or u > 2.0 ** -9 else (2.0 ** -25 * seen.double() @ v.abs()) / norm
    return o, u * o.abs() + (up + 2 * e) * a * (1 + 2 * u) + tiny + 1e-30


def attention(q, k, v, length: int, window: int, sinks: int, scale: float, two_terms: bool):
    """One sequence: q [new][q_heads][d], k, v [length][kv_heads][d] -> (o, bound) [new][q_heads][d]."""
    new, heads = q.shape[0], q.shape[1]
    group = heads // k.shape[1]
    seen = visible(range(length - new, length), length, window, sinks)
    o = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.full(q.shape, 1e-30, dtype=torch.float64)
    if length and new:
        for h in range(heads):
            o[:, h], bound[:, h] = rows(q[:, h], k[:, h // group], v[:, h // group], seen, scale, two_terms)
    return o, bound


class Cache:
    """Pages on `device` in which only the tokens given to `put` hold numbers: everything else is NaN,
    and table entries without a page are -1."""

    def __init__(self, kv_heads, dim, page, dtype, lengths, layers=1, layout="hnd", seed=1, spare=3, width=None,
                 device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        counts = [-(-n // page) for n in lengths]
        total = sum(counts) + spare
        if layout == "hnd":
            shape = (layers, total, kv_heads, page, dim)
            make = lambda: torch.full(shape, math.nan, dtype=dtype, device=device)  # noqa: E731
        elif layout == "nhd":
            shape = (layers, total, page, kv_heads, dim)
            make = lambda: torch.full(shape, math.nan, dtype=dtype, device=device).transpose(2, 3)  # noqa: E731
        else:  # gaps between the rows, pages outermost, layers inside
            make = lambda: torch.full((total, layers, kv_heads, page, dim + 24), math.nan, dtype=dtype,  # noqa: E731
                                      device=device)[..., 8:8 + dim].transpose(0, 1)
        self.k, self.v = make(), make()
        perm = torch.randperm(total, generator=gen)
        width = width or max([1] + counts) + 1
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        at = 0
        for s, c in enumerate(counts):
            self.table[s, :c] = perm[at:at + c].int()
            at += c
        self.spare = perm[at:].int()
        self.page, self.lengths = page, list(lengths)

    def where(self, seq, length=None):
        """(pages, rows) of a sequence's tokens."""
        j = torch.arange(self.lengths[seq] if length is None else length)
        return self.table[seq, j // self.page].long(), j % self.page

    def put(self, seq, k, v, layer=0, only=None):
        """k, v [length][kv_heads][dim] (CPU); only: which tokens."""
        pages, rows_ = self.where(seq)
        if only is not None:
            pages, rows_, k, v = pages[only], rows_[only], k[only], v[only]
        pages, rows_ = pages.to(self.k.device), rows_.to(self.k.device)
        self.k[layer, pages, :, rows_] = k.to(self.k)
        self.v[layer, pages, :, rows_] = v.to(self.v)

    def trim(self, seq, first, window, sinks):
        """Takes away the table's entries of pages that no query from position `first` on sees."""
        for slot in range(self.table.shape[1]):
            if (slot + 1) * self.page <= first - window + 1 and slot * self.page >= sinks:
                self.table[seq, slot] = -1
