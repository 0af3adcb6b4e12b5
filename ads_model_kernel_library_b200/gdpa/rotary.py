"""Queries and keys between a projection and the attention: the RMS norm of every head and its rotation by the token's position.

The reference takes its queries and keys as they are; its norms run over all heads of a token (:mod:`.megakernel`).  Here each head is normed by
itself and then rotated, in one pass over both tensors, with the gradient in another (``gdpa_qk_norm_rotary``, ``gdpa_qk_norm_rotary_bwd``).
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import paged

__all__ = ["qk_norm_rotary"]


def qk_norm_rotary(
    query: torch.Tensor,
    key: torch.Tensor,
    inv_freq: torch.Tensor,
    query_positions: torch.Tensor,
    key_positions: Optional[torch.Tensor] = None,
    query_weight: Optional[torch.Tensor] = None,
    key_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    norm: bool = True,
    interleaved: bool = False,
    sections: Optional[Sequence[int]] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Norm and rotate every head of ``query`` ``[total_q, H, D]`` and ``key`` ``[total_kv, H_kv, D]``; new contiguous tensors of their type.

    ``n = x * rsqrt(mean(x^2) + eps) * weight`` over the ``D`` values of a head (``weight`` ``[D]``, bf16 or fp32, ones if left out; ``norm=False``:
    ``n = x``), then pair ``i`` of the head turns by ``position * inv_freq[i]`` radians: the values ``i`` and ``i + len(inv_freq)``, with
    ``interleaved`` ``2 i`` and ``2 i + 1``.  ``inv_freq`` (fp32 or fp64, a multiple of 8 entries, ``D / 2`` at most) says how much of a head is rotated;
    the rest is only normed.  Angles are taken in 64 bits, so that far positions keep them; everything else in fp32, rounded once.

    Positions are int32 or int64 ``[tokens]``.  With ``sections`` (2 to 4 numbers that add up to ``len(inv_freq)``) they are ``[axes, tokens]``, and the
    first ``sections[0]`` pairs turn with the first axis, the next ``sections[1]`` with the second, and so on: time, height and width of images and video.
    ``key_positions`` are ``query_positions`` if left out (both tensors then have the same tokens).

    bf16 or fp32, head_dim 64 or 128, tokens and heads strided as in the attention (slices of a packed projection).  Gradients flow to query, key
    and the weights (``norm=False``: the weights take no part); their sums have an order that does not vary.  Not to ``inv_freq``.  Inputs with a
    tangent (forward-mode derivatives) are refused.
    """
    return (paged._operators or paged._load()).rotary(
        query, key, inv_freq, query_positions, query_positions if key_positions is None else key_positions, query_weight, key_weight, eps, norm, interleaved,
        () if sections is None else sections)
