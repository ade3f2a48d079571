"""Paged KV cache: K/V of sequences that grow token by token, and the attention of their newest tokens.

A pool of pages holds the rows of all sequences, ``[num_pages, page_size, H, D]`` for K and for V; row ``n`` of sequence
``b`` is row ``n % page_size`` of page ``block_table[b, n // page_size]``.  The operators take whole sequences
(``parallel_moda`` asks for ``T_q = T_kv * G``); this is what a generating program needs after the prompt:

    cache = PagedKVCache(num_pages, page_size, Hkv, D, dtype, device)           # one of each layer
    cache.append(k, v, block_table, seq_lens, lengths)                           # the prompt's K/V, after its attention
    ...
    depth = DepthKVCache(B, 1, n_layers - 1, Hkv, D, dtype, device)              # the new token's rows of earlier layers
    for layer in layers:                                                         # a decoding step
        q, k, v = ...                                                            # [B, G, H, D], [B, 1, H, D]
        o = layer.cache.decode(q, block_table, seq_lens, k, v, depth=depth, record=True, moda_group_num=G, rotary=rotary)
    seq_lens += 1

The functions do the same on tensors that the caller keeps; what they write counts as modified in place.  Nothing here synchronises or reads lengths on the host, so
that a step can be captured once and replayed while the sequences grow.  Rows that the tables or lengths
put outside the pool are left out and recorded (``moda_b200.device_status()``).  There is no backward: inputs
that require gradients are refused.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _cabi
from .depth_cache import DepthKVCache
from .rotary import Rotary


def paged_moda_append(k: torch.Tensor, v: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
                      block_table: torch.Tensor, seq_lens: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                      rotary: Optional[Rotary] = None) -> None:
    """Writes ``k, v [B, T, H, D]`` into the cache behind the ``seq_lens`` rows that the sequences hold.

    Token ``t`` of sequence ``b`` becomes row ``seq_lens[b] + t``, for ``t < lengths[b]`` (None: all of them).  With
    ``rotary`` keys are turned on the way, at their row's position.  ``block_table`` int32 ``[B, max_pages]``; ``seq_lens``,
    ``lengths`` int32 ``[B]``; ``seq_lens`` is not changed.  A ``lengths[b]`` below 0 or above ``T`` counts as 0 or
    ``T`` and is recorded (``device_status()``).  A page that is written to must belong to one sequence."""
    _cabi.native().paged_append(k, v, cache_k, cache_v, block_table, seq_lens, lengths, rotary)


def paged_moda_decode(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, block_table: torch.Tensor,
                      seq_lens: torch.Tensor, k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None,
                      cached_k: Optional[torch.Tensor] = None, cached_v: Optional[torch.Tensor] = None,
                      depth_positions: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                      moda_group_num: int = 1, rotary: Optional[Rotary] = None, need_lse: bool = False,
                      record_k: Optional[torch.Tensor] = None, record_v: Optional[torch.Tensor] = None, record_all: bool = False):
    """MoDA attention of one new token of each sequence: ``q [B, G, H, D]`` -> ``o [B, G, H, D]``, or ``(o, lse)`` with ``lse``
    fp32 ``[B, G, H]`` in base-2 units.

    The token sees the ``seq_lens[b]`` rows of its sequence in the cache, its own ``k, v [B, 1, H, D]`` where given (they are
    also appended, as by ``paged_moda_append``; without them its row is the sequence's last), and the depth rows
    ``cached_k, cached_v``: ``[B, L, H, D]`` of its own position, or ``[B, P, L, H, D]`` of positions of its chunk, of which it sees the
    first ``depth_positions[b]`` (int32; chunk-visible).  With ``rotary`` ``q`` and ``k`` are turned at the token's position:
    ``seq_lens[b]`` with ``k``, otherwise that of the sequence's last row (-1 where it has none, and sees depth rows alone); depth rows
    are used as they are.  ``record_k, record_v [B, 1, H, D]`` (none of the rows that are read) receive the token's row as
    written to the cache; a token whose row has no place there leaves them as they are, unless ``record_all``.  A token that sees
    nothing gets ``o = 0``, ``lse = -inf``."""
    r = _cabi.native().paged_decode(q, cache_k, cache_v, block_table, seq_lens, k, v, cached_k, cached_v, depth_positions, scale,
                                    moda_group_num, rotary, record_k, record_v, record_all)
    return r if need_lse else r[0]


class PagedKVCache:
    """The pages of one layer.  ``k`` and ``v`` are ``[num_pages, page_size, H, D]``; in memory a page holds its heads one after
    another, so that a head's rows of a page are one piece."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        assert num_pages >= 1 and page_size >= 1
        self.k, self.v = (torch.empty(num_pages, num_kv_heads, page_size, head_dim, dtype=dtype, device=device).transpose(1, 2)
                          for _ in range(2))

    def append(self, k, v, block_table, seq_lens, lengths=None, rotary=None) -> None:
        """``paged_moda_append`` into this layer's pages."""
        paged_moda_append(k, v, self.k, self.v, block_table, seq_lens, lengths, rotary)

    def decode(self, q, block_table, seq_lens, k=None, v=None, depth: Optional[DepthKVCache] = None, depth_positions=None,
               record: bool = False, scale=None, moda_group_num: int = 1, rotary=None, need_lse: bool = False):
        """``paged_moda_decode`` over this layer's pages and the layers that ``depth`` holds: a cache of one position, or (with
        ``depth_positions``) of the positions of a chunk.  ``record``: the token's row also becomes the next layer of ``depth``
        (of one position), for the layers after this one: also where it has no place in the pages, which leaves it out of this layer
        alone."""
        cached_k = cached_v = record_k = record_v = None
        if depth is not None:
            ck, cv = (x.view(depth.B, depth.T, depth.capacity, depth.H, depth.D) for x in (depth.k, depth.v))
            if depth.L > 0:
                cached_k, cached_v = ck[:, :, :depth.L], cv[:, :, :depth.L]
                if depth_positions is None:
                    assert depth.T == 1, "a depth cache of several positions needs depth_positions"
                    cached_k, cached_v = cached_k[:, 0], cached_v[:, 0]
        if record:
            assert depth is not None and depth.T == 1 and k is not None, "record needs k, v and a depth cache of one position"
            assert depth.L < depth.capacity, "DepthKVCache is full"
            record_k, record_v = ck[:, :, depth.L], cv[:, :, depth.L]
        r = paged_moda_decode(q, self.k, self.v, block_table, seq_lens, k, v, cached_k, cached_v,
                              depth_positions if cached_k is not None else None, scale, moda_group_num, rotary, need_lse, record_k, record_v, record)
        if record:
            depth.L += 1
        return r
