"""Serving over a paged KV cache held in 4 bits: block tables and slot maps built on the GPU,
quantise-and-append, read back, and causal sliding-window + global-token attention of new
tokens over the cache.

No counterpart in the reference, which attends to whole sequences only.  The functions take
the cache's tensors one by one; :class:`QuantizedKVCache` keeps them together.  Lengths, tables
and slots stay on the device and no call reads them on the host, so a serving step can be
captured into a CUDA graph and replayed.  The format of a pool is in include/lca.h.
"""
from __future__ import annotations

import math
import operator
from typing import NamedTuple, Sequence

import torch
from torch.autograd import forward_ad

from ._native import extension


class KVCacheStep(NamedTuple):
    """One step's placement (:func:`kv_cache_layout`), int32 tensors on the device."""

    slots: torch.Tensor       # [num_tokens] slot of each new token, -1 where there is none
    positions: torch.Tensor   # [num_tokens] position of each new token in its request, or -1
    cu_seqlens: torch.Tensor  # [batch + 1] row offsets of the requests
    kv_lens: torch.Tensor     # [batch] cached plus new tokens; 0 for a request that was not placed
    placed: torch.Tensor      # [batch] new tokens placed: new_lens, or 0
    seq_lens: torch.Tensor    # [batch] lengths after the step
    free_count: torch.Tensor  # [1] free pages after the step
    state: torch.Tensor       # [batch + 1] the two above as one tensor


def kv_cache_pool(num_pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A pool of ``num_pages`` pages: uint8 [num_pages, kv_heads, page_size, head_dim + 8], zeros.

    page_size is a multiple of 16, head_dim 64 or 128.  A token and head takes head_dim + 8
    bytes: 4 bits an element of K and V, and two 4-byte words of scale and zero point."""
    if page_size <= 0 or page_size % 16:
        raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    return torch.zeros(num_pages, kv_heads, page_size, head_dim + 8, dtype=torch.uint8, device=device)


def _need_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"long_context_attention: {what} must be a CUDA tensor on a B200 (sm_100a) GPU")


def _no_grad(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise NotImplementedError("long_context_attention: the operators of the 4-bit cache have no backward")
    # no tensor carries a forward-mode tangent outside a dual level, which is quicker to ask
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("long_context_attention: the operators of the 4-bit cache have no forward-mode derivative")


def kv_cache_layout(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor,
                    free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int,
                    num_tokens: int) -> KVCacheStep:
    """Places ``new_lens[b]`` tokens behind the ``seq_lens[b]`` cached ones of every request.

    block_table [batch, pages per request], seq_lens and new_lens [batch], free_pages [n] and
    free_count [1]: int32 CUDA tensors.  The new tokens of the requests are packed one request
    after the other into ``num_tokens`` rows (the capacity of a captured step; rows behind the
    last request get slot -1).  New pages are taken from the end of
    ``free_pages[:free_count]`` in request order and entered into block_table in place.  A request
    whose rows, table row or pages do not suffice is not placed at all: ``placed`` and ``kv_lens``
    are 0 for it, its slots -1, its length unchanged.  The lengths given stay as they are; the step
    holds the new ones.
    """
    _need_cuda(block_table, "block_table")
    return KVCacheStep(*extension().kv_cache_layout(block_table, seq_lens, new_lens, free_pages, free_count,
                                                    page_size, num_tokens))


def kv_cache_release(block_table: torch.Tensor, seq_lens: torch.Tensor, release: torch.Tensor,
                     free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int):
    """Puts the pages of the requests with ``release[b]`` (bool [batch]) back at the end of the free
    list, in place.  Returns ``(seq_lens, free_count, state)`` after it, as :class:`KVCacheStep` has
    them."""
    _need_cuda(block_table, "block_table")
    return tuple(extension().kv_cache_release(block_table, seq_lens, release, free_pages, free_count, page_size))


def kv_cache_append(pool: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises k, v [tokens, kv_heads, head_dim] (fp16 or bf16; any strides with a contiguous last
    dimension, such as slices of a fused projection) into ``slots`` of the pool, in place.  Slots
    outside the pool (-1) are skipped; the slots of one call are distinct."""
    _need_cuda(pool, "pool")
    _no_grad(k, v)
    extension().kv_cache_append(pool, k, v, slots)


def kv_cache_read(pool: torch.Tensor, slots: torch.Tensor, out_dtype: torch.dtype | None = None):
    """The values held in ``slots``: ``(k, v)``, each [tokens, kv_heads, head_dim] in ``out_dtype``
    (default float32).  A slot outside the pool reads as zeros."""
    _need_cuda(pool, "pool")
    return tuple(extension().kv_cache_read(pool, slots, out_dtype or torch.float32))


def sliding_window_attention_cached(
    Q: torch.Tensor,
    pool: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    window_size: int,
    global_tokens: Sequence[int] = (),
    scale: float | None = None,
    out_dtype: torch.dtype | None = None,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
):
    """Causal sliding-window + global-token attention of new tokens over a paged 4-bit cache.

    Q: [rows, heads, head_dim] fp16 or bf16 (last dimension contiguous, every row of a head on a
    16-byte boundary); request b's rows are
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` and are the last of its ``kv_lens[b]`` cached tokens.
    heads is a multiple of the pool's kv_heads.  The mask is that of ``sliding_window_attention(...,
    causal=True)``: key j is visible to the row at position p iff j <= p and (p - j <= window_size, or
    j or p is in ``global_tokens``, positions from 0 shared by the requests, at most 1024).  A
    window of the longest length or more is plain causal attention.  Returns O [rows, heads,
    head_dim] in ``out_dtype`` (default float32), and with ``return_lse`` also the natural-log LSE
    [heads, rows].  A row that sees nothing gets zeros and -inf.  Rows behind the last request are
    left as they were in ``out``; in the LSE, and in O without ``out``, they are not initialised.
    """
    _need_cuda(Q, "Q")
    _no_grad(Q) if out is None else _no_grad(Q, out)
    try:
        window_size = operator.index(window_size)
    except TypeError:
        raise TypeError("long_context_attention: attention over a cache takes one window_size, an int") from None
    if out_dtype is None:
        out_dtype = torch.float32 if out is None else out.dtype
    got = extension().sliding_window_attention_cached(
        Q, pool, block_table, kv_lens, cu_seqlens, window_size, list(global_tokens),
        1.0 / math.sqrt(Q.shape[-1]) if scale is None else scale, out_dtype, return_lse, out)
    return (got[0], got[1]) if return_lse else got[0]


class QuantizedKVCache:
    """A paged 4-bit KV cache of one attention layer for up to ``max_requests`` requests.

    A step of a serving loop::

        step = cache.reserve(new_lens, num_tokens)   # block table, slots, lengths, on the GPU
        cache.append(k, v, step)                     # the new tokens' keys and values
        o = cache.attention(q, step, window_size, global_tokens)
        cache.release(done)                          # pages of finished requests

    Every call runs on the current stream, allocates through torch's caching allocator and reads
    nothing on the host; a captured step advances the cache's state at each replay.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_requests: int,
                 max_pages_per_request: int | None = None, device="cuda"):
        self.pool = kv_cache_pool(num_pages, kv_heads, page_size, head_dim, device)
        self.page_size = page_size
        width = num_pages if max_pages_per_request is None else max_pages_per_request
        self.block_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self._state = torch.zeros(max_requests + 1, dtype=torch.int32, device=device)
        self._state[-1] = num_pages

    @property
    def seq_lens(self) -> torch.Tensor:
        """[max_requests] cached tokens of each request."""
        return self._state[:-1]

    @property
    def free_count(self) -> torch.Tensor:
        """[1] free pages."""
        return self._state[-1:]

    def reserve(self, new_lens: torch.Tensor, num_tokens: int) -> KVCacheStep:
        """Places new tokens (:func:`kv_cache_layout`) and advances the lengths and the free list."""
        step = kv_cache_layout(self.block_table, self.seq_lens, new_lens, self.free_pages, self.free_count,
                               self.page_size, num_tokens)
        self._state.copy_(step.state)
        return step

    def append(self, k: torch.Tensor, v: torch.Tensor, step: KVCacheStep) -> None:
        kv_cache_append(self.pool, k, v, step.slots)

    def attention(self, Q: torch.Tensor, step: KVCacheStep, window_size: int, global_tokens: Sequence[int] = (),
                  scale: float | None = None, **options):
        """:func:`sliding_window_attention_cached` of the step's tokens."""
        return sliding_window_attention_cached(Q, self.pool, self.block_table, step.kv_lens, step.cu_seqlens,
                                               window_size, global_tokens, scale, **options)

    def release(self, done: torch.Tensor) -> None:
        """Frees the pages of the requests with ``done[b]`` (bool [max_requests])."""
        _, _, state = kv_cache_release(self.block_table, self.seq_lens, done, self.free_pages, self.free_count,
                                       self.page_size)
        self._state.copy_(state)
