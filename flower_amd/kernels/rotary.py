"""Rotary positions of queries and keys, differentiable, on the HIP library (gfx950).

``apply_rotary(q, k, cos, sin, positions)`` turns the pairs of a head's first values by their token's angles, forward and
backward one HIP pass each (flw_rope; the checks and the autograd node are native code). The reference's RotaryEmbedding (flower/models/base.py:436-483) turns whole heads,
pairs next to each other, at positions 0 .. T - 1; here the pairs may also be half a rotation apart ("half"), the tables
may cover only the first part of the head, and each token has a position of its own. Tables are made by
``flower_amd.attention.rotary_tables`` (or ``RotaryEmbedding.pair_tables``), which also scales them for long contexts.
"""

from __future__ import annotations

import torch

from .. import _lib

ROTARY_LAYOUTS = ("interleaved", "half")


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor | None = None, *, layout: str = "interleaved"):
    """(q', k') of q (B, H, T, D) and k (B, KV, T, D) (or None), bf16 or fp32, contiguous (B, heads, T, D).

    The first R = 2 * cos.shape[1] values of each head are pairs (a, b), (2 i, 2 i + 1) ("interleaved") or (i, i + R / 2)
    ("half"), and become (a c - b s, b c + a s) with c = cos[position, i], s = sin[position, i]; the rest of the head is
    copied. cos, sin: fp32 [positions, R / 2]. positions: int32 or int64 (T,) or (B, T); None is 0 .. T - 1. A position
    outside the tables makes that token's pairs NaN. fp32 arithmetic, rounded once to q's dtype. Differentiable in q
    and k by backward, also twice; tensors with a forward-mode tangent are refused.
    """
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"layout must be one of {ROTARY_LAYOUTS}, got {layout!r}")
    return _lib.native().apply_rotary(q, k, cos, sin, positions, layout == "half", _lib.stream_or_none(q))


__all__ = ["apply_rotary", "ROTARY_LAYOUTS"]
