"""Rotary positions of queries and keys, in the operators' folded layout.

    inv_freq, scale = rotary_frequencies(D, base=10000.0, device=q.device)
    rotary = Rotary(inv_freq, interleaved=False, scale=scale)
    q, k = rotary_embedding(q, k, rotary, moda_group_num=G)        # q [B, T*G, H, D], k [B, T, H, D]
    o = parallel_moda(q, k, v, ..., moda_group_num=G)

Row ``t*G + g`` of a folded ``q`` stands at position ``t``, so a rotation written for ``[B, T, heads, D]`` cannot
be used on it without unfolding.  Angles are reduced in whole numbers (``csrc/rotary_kernels.cuh``): far positions are as
exact as near ones, and there are no tables to build or to outgrow.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _cabi


class Rotary(NamedTuple):
    """How vectors turn with their position.

    inv_freq     float64 ``[rotary_dim / 2]`` on the tensors' device: radians a position of each pair.  rotary_dim, a
                 multiple of 16 of at most the head dim, is how much of a head turns (its first elements)
    interleaved  pairs ``(2i, 2i+1)`` instead of ``(i, i + rotary_dim / 2)``
    scale        factor on the turned elements
    """
    inv_freq: torch.Tensor
    interleaved: bool = False
    scale: float = 1.0


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, scale)`` for ``Rotary``: ``base ** (-2i / rotary_dim)``, stretched for contexts ``factor`` times longer.

    scaling  None      as it is
             "linear"  positions divided by ``factor`` (every frequency divided by it)
             "ntk"     the base grown by ``factor ** (rotary_dim / (rotary_dim - 2))``: the slowest pair as under "linear",
                       the fastest as it is
             "yarn"    pairs that turn more than ``beta_fast`` times over ``original_length`` positions as they are, those
                       that turn less than ``beta_slow`` times as under "linear", a linear ramp between, and vectors grown by
                       ``0.1 ln(factor) + 1``
    """
    assert rotary_dim >= 16 and rotary_dim % 16 == 0, "rotary_dim must be a positive multiple of 16"
    assert factor > 0 and base > 0
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv_freq = base ** (-2.0 * i / rotary_dim)
    scale = 1.0
    if scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "yarn":
        assert original_length is not None and original_length > 0, "yarn needs original_length"
        assert base > 1 and 0 < beta_slow < beta_fast

        def pair_that_turns(times):
            return rotary_dim * math.log(original_length / (times * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_that_turns(beta_fast)), 0)
        high = min(math.ceil(pair_that_turns(beta_slow)), rotary_dim - 1)
        slow = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv_freq = inv_freq * (1 - slow) + inv_freq / factor * slow
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    else:
        assert scaling in (None, "ntk"), "scaling must be None, 'linear', 'ntk' or 'yarn'"
    return inv_freq.to(device), scale


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], rotary: Rotary,
                     positions: Union[None, int, torch.Tensor] = None, moda_group_num: int = 1):
    """Turns ``q [B, T*moda_group_num, H, D]`` and ``k [B, T, H, D]`` by their positions: ``(q, k)``, or ``q`` where ``k`` is None.

    ``positions``: None (token ``t`` stands at ``t``), the first token's position, or an int32 / int64 tensor ``[T]`` or
    ``[B, T]``.  Differentiable in ``q`` and ``k``; positions and frequencies are used again in the backward, which
    notices if they have been changed in between."""
    q, k = _cabi.native().rotary(q, k, rotary, positions, moda_group_num)
    return q if k is None else (q, k)
