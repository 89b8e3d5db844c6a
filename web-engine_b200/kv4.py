"""A paged 4-bit K/V cache and the attention of newest tokens over it (we_kv4_*; no reference counterpart).

A step of a decoding loop, for every layer: ``append`` the step's k and v rows, then ``attention`` of the step's
queries over the cache; after the last layer ``advance`` the lengths once. ``unpack`` gives rows back as f32 or bf16
(a prompt's own attention, or a look into the cache). The ``*_call`` forms convert their arguments once and are then
called every token (kernels.Call).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from . import _lib as L
from .graph import Graph, addr
from .kernels import Call

GROUP = 64  # values that share one f16 scale


@dataclass
class Cache:
    """One layer's cache, as device buffers: codes k, v [pages, kv_heads, page, dim / 2] (int4, low nibble = even
    value), f16 scales [pages, kv_heads, page, dim / 64], page_table int32 [batch, max_pages] and lengths int32 [batch]
    (tokens before the step; negative: idle). Layers of one model share page_table and lengths. dim 64, 128 or 256;
    page a multiple of 16."""

    k: object
    v: object
    k_scale: object
    v_scale: object
    page_table: object
    lengths: object
    pages: int
    max_pages: int
    batch: int
    kv_heads: int
    page: int
    dim: int

    @classmethod
    def create(cls, graph: Graph, batch: int, tokens: int, kv_heads: int, dim: int, page: int = 64,
               like: "Cache | None" = None) -> "Cache":
        """An empty cache with room for `tokens` tokens of each sequence: sequence b owns pages b * max_pages and on.
        `like`: another layer's cache, whose page table and lengths this one shares."""
        per = -(-tokens // page)
        rows = batch * per * kv_heads * page
        if like is not None:
            if (like.batch, like.max_pages, like.page) != (batch, per, page):
                raise ValueError("layers that share a page table have the same batch, tokens and page")
            table, lengths = like.page_table, like.lengths
        else:
            table = graph.buffer(np.arange(batch * per, dtype=np.int32))
            lengths = graph.buffer(np.zeros(batch, np.int32))
        return cls(graph.buffer(rows * dim // 2), graph.buffer(rows * dim // 2), graph.buffer(rows * dim // GROUP * 2),
                   graph.buffer(rows * dim // GROUP * 2), table, lengths, batch * per, per, batch, kv_heads, page, dim)

    def desc(self) -> L.KV4Desc:
        return L.KV4Desc(*(addr(b).value for b in (self.k, self.v, self.k_scale, self.v_scale, self.page_table,
                                                   self.lengths)),
                         self.pages, self.max_pages, self.batch, self.kv_heads, self.page, self.dim)


def append_call(graph: Graph, cache: Cache, k, v, tokens: int, dtype: str = "bf16", stride: int = 0) -> Call:
    """The prepared form of `append`."""
    d = cache.desc()
    return Call(graph, L.lib().we_kv4_append, (C.pointer(d), addr(k), addr(v), L.DTYPES[dtype], tokens, stride),
                (d, cache, k, v))


def append(graph: Graph, cache: Cache, k, v, tokens: int, dtype: str = "bf16", stride: int = 0) -> None:
    """Quantises k, v [batch, tokens, kv_heads, dim] (`stride` values from a token to the next, 0 = contiguous) into
    each sequence's rows lengths[b] .. lengths[b] + tokens - 1."""
    append_call(graph, cache, k, v, tokens, dtype, stride)()


def unpack_call(graph: Graph, cache: Cache, k, v, tokens: int, dtype: str = "bf16", start=None) -> Call:
    """The prepared form of `unpack`."""
    d = cache.desc()
    return Call(graph, L.lib().we_kv4_unpack, (C.pointer(d), addr(k), addr(v), L.DTYPES[dtype], tokens, addr(start)),
                (d, cache, k, v, start))


def unpack(graph: Graph, cache: Cache, k, v, tokens: int, dtype: str = "bf16", start=None) -> None:
    """Writes the values of rows start[b] .. start[b] + tokens - 1 (int32 [batch] on the device; None: lengths[b] on,
    the rows of the step's append) to k, v [batch, tokens, kv_heads, dim]. k or v may be None."""
    unpack_call(graph, cache, k, v, tokens, dtype, start)()


def attention_call(graph: Graph, cache: Cache, q, out, tokens: int, heads: int, dtype: str = "bf16",
                   out_dtype: str = "bf16", q_stride: int = 0, out_stride: int = 0, scale: float = 0.0) -> Call:
    """The prepared form of `attention`."""
    d = cache.desc()
    return Call(graph, L.lib().we_kv4_attention, (C.pointer(d), addr(q), L.DTYPES[dtype], tokens, heads, q_stride, scale,
                                                  addr(out), L.DTYPES[out_dtype], out_stride), (d, cache, q, out))


def attention(graph: Graph, cache: Cache, q, out, tokens: int, heads: int, dtype: str = "bf16", out_dtype: str = "bf16",
              q_stride: int = 0, out_stride: int = 0, scale: float = 0.0) -> None:
    """softmax(scale q k^T) v of each sequence's newest tokens over its cache: q, out [batch, tokens, heads, dim]; query i
    sees keys 0 .. lengths[b] + i (appended before). scale 0 = 1 / sqrt(dim), else of either sign. Idle sequences give
    zeros; a group of 64 values that held a NaN when it was appended gives NaN."""
    attention_call(graph, cache, q, out, tokens, heads, dtype, out_dtype, q_stride, out_stride, scale)()


def advance_call(graph: Graph, cache: Cache, tokens: int = 1) -> Call:
    """The prepared form of `advance`."""
    d = cache.desc()
    return Call(graph, L.lib().we_kv4_advance, (C.pointer(d), tokens), (d, cache))


def advance(graph: Graph, cache: Cache, tokens: int = 1) -> None:
    """lengths[b] += tokens for every sequence that is not idle: once per step, after the last layer."""
    advance_call(graph, cache, tokens)()
