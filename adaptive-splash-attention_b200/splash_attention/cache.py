"""Serving from a 4-bit paged key/value cache.

A model trained with this package's attention is served from a pool of pages
that hold keys and values in 4 bits (5 with their scales): ``cache_write``
quantises new tokens into it, ``cache_attention`` attends over it with softmax
or the α-entmax weights of training, ``select_pages`` chooses the pages a query
reads by a cheap score of the pages' bounds, and ``cache_read`` and
``cache_bounds`` read it back.  The formats are described in include/asa.h.
Every computation runs in hand-written CUDA kernels behind the C ABI; the calls
go on the current stream, synchronise nothing, can be captured in CUDA graphs and
carry no gradients.  The reference has no counterpart.

Index tensors (block tables, lengths, starts, counts, page lists) are int32 on
the cache's device; other integer types are converted.  Positions past the
block table and page ids outside the pool (whole numbers that int32 does not hold
among them) are neither read nor written, and record an error that
``device_error()`` reads; the training operators do not see it.
"""
from typing import NamedTuple

import torch

# (the overloads themselves: a step makes these calls once a layer)
_ops = torch.ops.splash_attention
_cache_write, _cache_read, _cache_bounds = (getattr(_ops, n).default for n in ("cache_write", "cache_read", "cache_bounds"))
_cache_select, _cache_attention = _ops.cache_select.default, _ops.cache_attention.default

BOUNDS_PAD = 16
HEAD_DIMS = (32, 64, 96, 128)
PAGE_SIZES = (16, 32, 64, 128)


class KVCache(NamedTuple):
    """The two tensors of a cache: ``pool`` uint8 [pages, kv_heads, record] and
    ``bounds`` int8 [pages, kv_heads, 2 head_dim + 16]."""
    pool: torch.Tensor
    bounds: torch.Tensor

    @property
    def head_dim(self):
        return (self.bounds.shape[-1] - BOUNDS_PAD) // 2

    @property
    def page_size(self):
        return self.pool.shape[-1] * 4 // (5 * self.head_dim)

    @property
    def kv_heads(self):
        return self.pool.shape[1]


def new_cache(num_pages, kv_heads, head_dim, page_size=64, device="cuda"):
    """An empty cache of ``num_pages`` pages of ``page_size`` tokens."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"splash_attention: a cache's head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"splash_attention: page_size must be one of {PAGE_SIZES}, got {page_size}")
    if num_pages < 0 or kv_heads < 1:
        raise ValueError("splash_attention: a cache has at least one key head and no negative number of pages")
    return KVCache(torch.zeros(num_pages, kv_heads, page_size * head_dim * 5 // 4, dtype=torch.uint8, device=device),
                   torch.zeros(num_pages, kv_heads, 2 * head_dim + BOUNDS_PAD, dtype=torch.int8, device=device))


def cache_write(K, V, cache, block_table, start, count=None):
    """Quantises K and V [B, T, kv_heads, head_dim] (bfloat16 or float32, any
    strides) into the cache: sequence b's first ``count[b]`` tokens (all T without
    ``count``) at positions start[b], start[b] + 1, ... of its ``block_table`` row.
    A page belongs to one sequence; its bounds start over when its first slot is
    written, and otherwise grow."""
    _cache_write(K, V, cache.pool, cache.bounds, block_table, start, count)


def cache_read(cache, block_table, start, T, count=None, *, dtype=torch.bfloat16):
    """Reads positions start[b] .. start[b] + T - 1 back: (K, V)
    [B, T, kv_heads, head_dim] bfloat16 or float32, zero from ``count[b]`` on."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"splash_attention: unsupported dtype {dtype} (float32 or bfloat16)")
    return _cache_read(cache.pool, cache.bounds, block_table, start, T, count, dtype == torch.float32)


def cache_bounds(cache, pages):
    """The bounds of the pool's pages ``pages`` [n] as values: (upper, lower)
    float32 [n, kv_heads, head_dim], no channel's keys, as they were given, above or
    below them (what is read back has been rounded, and may lie outside)."""
    return _cache_bounds(cache.bounds, pages)


def select_pages(q, cache, block_table, lengths, keep):
    """The ``keep`` pages that each query and key head should read: int32
    [B, T, kv_heads, keep], ascending places in the block table row, -1 behind
    the last.  q: [B, T, heads, head_dim] bfloat16; query t of sequence b stands
    at position lengths[b] - T + t.  Its own page is always among them; the others
    score highest by an upper bound of q.k from their bounds, q rounded to 8 bits (so a
    page may score a little below its best key), the largest over the heads that
    share the key head, ties to the earlier page."""
    return _cache_select(q, cache.pool, cache.bounds, block_table, lengths, keep)


def cache_attention(q, cache, block_table, lengths, *, sm_scale=None, alpha=1.0, pages=None):
    """Attention of q [B, T, heads, head_dim] bfloat16 over the cache: [B, T,
    heads, head_dim] bfloat16.  ``lengths[b]`` counts sequence b's tokens, the T of
    this call (written before) among them: query t stands at position
    lengths[b] - T + t and sees the keys up to its own.  ``heads`` is any multiple of
    the cache's heads; query heads g * i .. g * i + g - 1 share key head i.

    ``alpha`` 1 gives softmax weights; 1.05 to 3 the exact α-entmax weights of
    ``splash_attention(tau_mode="exact", ref_tile_load=False)``, scores clamped to ±10
    as in training.  ``pages`` (from ``select_pages``: no page twice) restricts each
    query to the listed pages.  A query that sees no key gives zeros, one holding a
    NaN or an infinity NaN.  Weights are held in 11 bits; softmax over 64 and more query
    rows a key head (T * heads / kv_heads, head_dim 64 or 128, no ``pages``) also holds
    keys, less their group's middle, and values in 11 bits."""
    if sm_scale is None:
        sm_scale = q.shape[-1] ** -0.5
    return _cache_attention(q, cache.pool, cache.bounds, block_table, lengths, pages, sm_scale, alpha)
