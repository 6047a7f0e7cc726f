"""The attention between two linear calls of a layer, on the protocol's numbers.

A ``private_matrix`` call ends in ring-59 words: fixed-point values with a known number of fraction
bits, modulo 2^59.  Where one party holds the decoded q/k/v product (a client that computes the
non-linear steps itself, or a check of the protocol in the clear), ``RingAttention`` takes those
words, keeps the keys and values in a ``KvCache``, and returns the attention as ring-59 words for
the o call.  In between everything is 16-bit floating point with 32-bit sums: it is not the
reference's exact-integer attention, which runs as a two-party protocol and is out of this
library's scope.

Norms of the heads and rotary positions, as a Qwen3 layer has them between the call and the attention, are applied on
the way into the cache where ``rotary`` and the norms' weights are given; without them it is the attention alone, on q and
k as the call leaves them.

    att = RingAttention(ctx, q_heads=16, kv_heads=8, dim=128, fraction=24, out_fraction=12, pages=4096,
                        rotary=Rotary(ctx, 128, base=1e6), share=True)
    doc = att.open()
    att.extend({doc: 512})                      # a retrieved document
    o_words = att.layer(qkv_words)              # [512][4096] -> [512][2048]
    answers = att.fork(doc, 4)                  # four answers share its pages (and with share read them once)
    att.extend({a: 1 for a in answers})         # one token each
    o_words = att.layer(qkv_words_of_the_step)  # [4][4096] -> [4][2048], rows in the cache's order
"""
from __future__ import annotations

from .backend import Context
from .kvcache import KvCache
from .layout import MASK59

_HALF = 1 << 58


def words_to_floats(torch, words, fraction: int):
    """int64 ring-59 words -> their centred values as float32 (the nearest)."""
    centred = ((words + _HALF) & MASK59) - _HALF
    return (centred.double() * 2.0 ** -fraction).float()


def floats_to_words(torch, x, fraction: int):
    """The nearest fixed-point values (ties to even) as int64 ring-59 words; the values have to lie
    within +-2^(58 - fraction)."""
    return torch.round(x.double() * 2.0 ** fraction).long() & MASK59


class RingAttention:
    """Keys, values and attention of `layers` layers for a set of sequences.  qkv words of a call are
    [tokens][(q_heads + 2 kv_heads) dim], q first, with `fraction` fraction bits; the result has
    `out_fraction`.  window and sinks as for ``PagedKv.decode``.  rotary: a ``Rotary`` for queries and keys; q_norm, k_norm:
    float32 weights [dim], of each layer [layers][dim], of the norm of each head before it (eps).  share: rows that share
    their first pages read them once together (``KvCache.attend``)."""

    def __init__(self, ctx: Context, q_heads: int, kv_heads: int, dim: int, fraction: int, out_fraction: int, pages: int,
                 layers: int = 1, page_tokens: int = 16, sequences: int = 64, tokens: int = 4096, dtype=None,
                 window: int = 0, sinks: int = 0, rotary=None, q_norm=None, k_norm=None, eps: float = 1e-6, share: bool = False):
        import torch
        if rotary is None and (q_norm is not None or k_norm is not None):
            raise ValueError("E_ROTARY_NORM: norms of the heads come with a rotation")
        for w in (q_norm, k_norm):
            if w is not None and tuple(w.shape) not in ((dim,), (layers, dim)):
                raise ValueError("E_ROTARY_SHAPE: a norm has weights [dim] or [layers][dim]")
        if not 0 <= fraction <= 58 or not 0 <= out_fraction <= 58:
            raise ValueError("E_SHAPE")
        self._torch = torch
        self.q_heads, self.kv_heads, self.dim = q_heads, kv_heads, dim
        self.fraction, self.out_fraction, self.window, self.sinks = fraction, out_fraction, window, sinks
        self.rotary, self.q_norm, self.k_norm, self.eps, self.share = rotary, q_norm, k_norm, eps, share
        self.cache = KvCache(ctx, pages, kv_heads, dim, layers, page_tokens, sequences, tokens, dtype)
        self.open, self.free, self.fork, self.compact = (self.cache.open, self.cache.free, self.cache.fork,
                                                         self.cache.compact)

    def extend(self, counts: dict[int, int]) -> None:
        """Begins a step: counts[row] new tokens for each row.  Pages that no later query sees are given
        up first."""
        if self.window:
            self.cache.trim(self.window, self.sinks)
        self.cache.extend(counts)

    def layer(self, qkv_words, layer: int = 0):
        """One layer of the step: int64 words [tokens][(q_heads + 2 kv_heads) dim] -> [tokens][q_heads dim]."""
        h, g, d = self.q_heads, self.kv_heads, self.dim
        if qkv_words.dim() != 2 or qkv_words.shape[1] != (h + 2 * g) * d:
            raise ValueError("E_SHAPE")
        x = words_to_floats(self._torch, qkv_words, self.fraction).unflatten(1, (h + 2 * g, d))
        if self.rotary is None:
            self.cache.append(x[:, h:h + g], x[:, h + g:], layer)
            q = x[:, :h].to(self.cache.kv.k.dtype)
        else:
            of_layer = lambda w: w if w is None or w.dim() == 1 else w[layer]  # noqa: E731
            q = self.cache.append_rotary(x[:, h:h + g], x[:, h + g:], self.rotary, x[:, :h], of_layer(self.q_norm),
                                         of_layer(self.k_norm), self.eps, layer)
        out = self.cache.attend(q, layer, self.window, self.sinks, share=self.share)
        return floats_to_words(self._torch, out.flatten(1), self.out_fraction)
