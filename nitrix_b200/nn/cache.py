"""A paged key / value cache, in the operands' type or in 4 or 8 bits, and the attention of one new token per sequence over it
(``include/nitrix_b200_cache.h``).

The cache of a layer is a pool of pages and a table that says which pages hold which sequence's tokens.  All bookkeeping runs
on the device: no call waits for the GPU, and a generation step can be captured into a CUDA graph.

A :class:`PagedCache` or :class:`QuantizedCache` is a value: each function takes one and returns the next.  Pages are shared between
them and written in place, but a call only writes slots that are free in the cache that it is given.  The cache given therefore
stays valid (a step that turns out wrong is undone by going on from the earlier value) until another call writes pages.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, TypeVar, Union

import torch

from .. import _cabi
from ..backend import resolve_backend
from .attention import default_scale

__all__ = ["PagedCache", "paged_cache", "QuantizedCache", "quantized_cache", "cache_append", "cache_fork", "cache_free", "cache_compact",
           "cache_read", "decode_attention"]


class PagedCache(NamedTuple):
    """Pages of ``k`` and ``v``, ``(pages, key heads, page size, head dim)``, and the int32 arrays that describe their use."""

    k_pages: torch.Tensor
    v_pages: torch.Tensor
    table: torch.Tensor         #: (sequences, width): the pages of each sequence in order
    lengths: torch.Tensor       #: (sequences,): tokens of each sequence
    free_pages: torch.Tensor    #: (pages,): of which free_range[0] .. free_range[1] are free, in the order of their use
    free_range: torch.Tensor    #: (2,)
    shortfall: torch.Tensor     #: (1,): tokens that the last call had no page for and dropped


class QuantizedCache(NamedTuple):
    """Pages of codes of ``k`` and ``v`` with a step for each 32 elements, and the int32 arrays of :class:`PagedCache`.

    A value is ``step * (code - 2 ** (bits - 1))``.  The step of a group, fp16, is the one that gives its element of largest
    magnitude the code 0 (magnitudes over 524032 in 4 bits, 8384512 in 8, are cut to that; a group with a NaN or an infinity reads
    as NaN).  A row of codes is ``(8, groups, bits / 2)`` bytes: of every group the elements ``4 j .. 4 j + 3`` lie together, the first
    in the lowest bits."""

    k_codes: torch.Tensor       #: uint8 (pages, key heads, page size, head dim * bits / 8)
    v_codes: torch.Tensor
    k_steps: torch.Tensor       #: float16 (pages, key heads, page size, head dim / 32)
    v_steps: torch.Tensor
    table: torch.Tensor
    lengths: torch.Tensor
    free_pages: torch.Tensor
    free_range: torch.Tensor
    shortfall: torch.Tensor


Cache = TypeVar("Cache", PagedCache, QuantizedCache)


def _parts(cache):
    """``(pages, table .. shortfall, steps)``: what the operators take in this order."""
    if isinstance(cache, QuantizedCache):
        return cache[:2], cache[4:], cache[2:4]
    return cache[:2], cache[2:], (None, None)


def _state(pages: int, page_size: int, sequences: int, max_length: int, device):
    ints = dict(dtype=torch.int32, device=device)
    return (torch.full((sequences, -(-max_length // page_size)), -1, **ints), torch.zeros(sequences, **ints), torch.arange(pages, **ints),
            torch.tensor([0, pages], **ints), torch.zeros(1, **ints))


def paged_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, *, sequences: int, max_length: int,
                dtype: torch.dtype = torch.bfloat16, device="cuda") -> PagedCache:
    """An empty cache for ``sequences`` sequences of up to ``max_length`` tokens."""
    for name, value in dict(pages=pages, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim, max_length=max_length).items():
        if value < 1:
            raise ValueError(f"paged_cache: {name} must be positive; got {value}")
    shape = (pages, kv_heads, page_size, head_dim)
    return PagedCache(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                      *_state(pages, page_size, sequences, max_length, device))


def quantized_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, *, bits: int = 4, sequences: int, max_length: int,
                    device="cuda") -> QuantizedCache:
    """An empty cache in 4 or 8 bits for ``sequences`` sequences of up to ``max_length`` tokens; ``head_dim`` is a multiple of 32."""
    for name, value in dict(pages=pages, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim, max_length=max_length).items():
        if value < 1:
            raise ValueError(f"quantized_cache: {name} must be positive; got {value}")
    if bits not in (4, 8):
        raise ValueError(f"quantized_cache: bits must be 4 or 8; got {bits}")
    if head_dim % 32:
        raise ValueError(f"quantized_cache: head_dim must be a multiple of 32; got {head_dim}")
    rows = (pages, kv_heads, page_size)
    codes = [torch.zeros(*rows, head_dim * bits // 8, dtype=torch.uint8, device=device) for _ in range(2)]
    steps = [torch.zeros(*rows, head_dim // 32, dtype=torch.float16, device=device) for _ in range(2)]
    return QuantizedCache(*codes, *steps, *_state(pages, page_size, sequences, max_length, device))


def cache_append(cache: Cache, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, *, backend: str = "auto") -> Cache:
    """The cache with tokens ``offsets[i] .. offsets[i + 1]`` of ``k`` and ``v`` ``(tokens, key heads, head dim)`` behind those
    of sequence ``i``; ``offsets`` is int32 ``(sequences + 1,)``.  New pages go to the sequences in order.  Tokens for which
    there is no page (or no room in the table) are dropped from the end of a sequence and counted in ``shortfall``, as are those
    that offsets name beyond ``k`` and ``v``; offsets that descend store nothing.  A :class:`PagedCache` takes its own dtype, a
    :class:`QuantizedCache` quantises fp32, bf16 or fp16.  The cache holds values: no gradient flows back through it."""
    resolve_backend(backend)
    pages, state, steps = _parts(cache)
    lengths, free_range, shortfall = _cabi.torch_ops().cache_append(*pages, *state[:4], k, v, offsets, *steps)
    return cache._replace(lengths=lengths, free_range=free_range, shortfall=shortfall)


def _forked(cache: Cache, rows: torch.Tensor, finished: bool) -> Cache:
    pages, state, steps = _parts(cache)
    table, lengths, free_pages, free_range, shortfall = _cabi.torch_ops().cache_fork(*pages, *state[:4], rows, finished, *steps)
    return cache._replace(table=table, lengths=lengths, free_pages=free_pages, free_range=free_range, shortfall=shortfall)


def cache_fork(cache: Cache, parents: torch.Tensor, *, backend: str = "auto") -> Cache:
    """The cache whose sequence ``i`` is a copy of sequence ``parents[i]`` (int32; any number of them; a negative one leaves
    the row empty).  Full pages are shared; the page that is still being filled is copied for every child but the first.  Pages
    that no sequence reaches any more are free; the list of free pages is then in ascending order."""
    resolve_backend(backend)
    return _forked(cache, parents, False)


def cache_free(cache: Cache, finished: torch.Tensor, *, backend: str = "auto") -> Cache:
    """The cache without the sequences that ``finished`` (bool, ``(sequences,)``) names: their rows are empty."""
    resolve_backend(backend)
    return _forked(cache, finished, True)


def cache_compact(cache: Cache, *, backend: str = "auto") -> Cache:
    """The cache with its live pages at the front of the pool: those behind move to the lowest free places, in order."""
    resolve_backend(backend)
    pages, state, steps = _parts(cache)
    table, free_pages, free_range, shortfall = _cabi.torch_ops().cache_compact(*pages, *state[:4], *steps)
    return cache._replace(table=table, free_pages=free_pages, free_range=free_range, shortfall=shortfall)


def cache_read(cache: Union[PagedCache, QuantizedCache], offsets: torch.Tensor, tokens: int, *, starts: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None, backend: str = "auto") -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens of the cache as packed rows ``(k, v)``, each ``(tokens, key heads, head dim)``.

    Rows ``offsets[i] .. offsets[i + 1]`` (int32, ``(sequences + 1,)``, not descending) are the tokens of sequence ``i`` from its
    position ``starts[i]`` on (int32; the first one by default); rows of no sequence, and those of positions that the sequence does
    not hold, are zeros.  With offsets that are the sums of ``cache.lengths`` these are the keys and values of
    :func:`packed_attention` for the next chunk of every prompt.  ``dtype`` is what a :class:`QuantizedCache` is read as (bf16 by
    default); a :class:`PagedCache` has its own.  Not differentiable."""
    resolve_backend(backend)
    pages, state, steps = _parts(cache)
    return _cabi.torch_ops().cache_read(*pages, *state[:2], offsets, starts, tokens, dtype, *steps)


def decode_attention(q: torch.Tensor, cache: Union[PagedCache, QuantizedCache], *, scale: Optional[float] = None,
                     backend: str = "auto") -> torch.Tensor:
    """Attention of one query token per sequence, ``q`` ``(sequences, heads, head dim)``, over the sequence's tokens in the
    cache (the new token's own among them, once it has been appended).  Query head ``h`` reads key head
    ``h // (heads // key heads)``; an empty sequence gives zeros.  ``q`` has the dtype of a :class:`PagedCache`; a
    :class:`QuantizedCache` takes fp32, bf16 or fp16.  Not differentiable."""
    resolve_backend(backend)
    pages, state, steps = _parts(cache)
    return _cabi.torch_ops().decode_attention(q, *pages, *state[:2], default_scale(q.shape[-1]) if scale is None else float(scale), *steps)
