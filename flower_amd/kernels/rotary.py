"""Rotary positions of queries and keys, differentiable, on the HIP library (gfx950).

``apply_rotary(q, k, cos, sin, positions)`` turns the pairs of a head's first values by their token's angles, forward and
backward one HIP pass each (flw_rope). The reference's RotaryEmbedding (flower/models/base.py:436-483) turns whole heads,
pairs next to each other, at positions 0 .. T - 1; here the pairs may also be half a rotation apart ("half"), the tables
may cover only the first part of the head, and each token has a position of its own. Tables are made by
``flower_amd.attention.rotary_tables`` (or ``RotaryEmbedding.pair_tables``), which also scales them for long contexts.
"""

from __future__ import annotations

import torch

from .. import _lib

ROTARY_LAYOUTS = ("interleaved", "half")


class _Rotary(torch.autograd.Function):
    """The rotation is linear, its gradient the opposite rotation of the gradient: the node is its own backward."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, half, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.half, ctx.inverse = half, inverse
        ctx.set_materialize_grads(False)
        return _lib.native().rope(q, k, cos, sin, positions, half, inverse, _lib.stream_of(q))

    @staticmethod
    def backward(ctx, gq, gk):
        cos, sin, positions = ctx.saved_tensors
        if gq is None and gk is None:
            return (None,) * 7
        if gq is None:
            gk, _ = _Rotary.apply(gk, None, cos, sin, positions, ctx.half, not ctx.inverse)
        else:
            gq, gk = _Rotary.apply(gq, gk, cos, sin, positions, ctx.half, not ctx.inverse)
        return gq, gk, None, None, None, None, None


def check_tables(cos: torch.Tensor, sin: torch.Tensor, head_dim: int, layout: str, device) -> None:
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"layout must be one of {ROTARY_LAYOUTS}, got {layout!r}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 [positions, rotary_dim / 2] tables of one shape, got "
                         f"{tuple(cos.shape)} {cos.dtype} and {tuple(sin.shape)} {sin.dtype}")
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous")
    if 2 * cos.shape[1] > head_dim or cos.shape[1] % 4 or cos.shape[1] == 0:
        raise ValueError(f"rotary_dim must be a multiple of 8 up to the head_dim {head_dim}, got {2 * cos.shape[1]}")
    if cos.device != device or sin.device != device:
        raise ValueError(f"cos and sin must be on {device}")


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor | None = None, *, layout: str = "interleaved"):
    """(q', k') of q (B, H, T, D) and k (B, KV, T, D) (or None), bf16 or fp32, contiguous (B, heads, T, D).

    The first R = 2 * cos.shape[1] values of each head are pairs (a, b), (2 i, 2 i + 1) ("interleaved") or (i, i + R / 2)
    ("half"), and become (a c - b s, b c + a s) with c = cos[position, i], s = sin[position, i]; the rest of the head is
    copied. cos, sin: fp32 [positions, R / 2]. positions: int32 or int64 (T,) or (B, T); None is 0 .. T - 1. A position
    outside the tables makes that token's pairs NaN. fp32 arithmetic, rounded once to q's dtype. Differentiable in q and k.
    """
    x = (q,) if k is None else (q, k)
    if any(t.dim() != 4 for t in x):
        raise ValueError(f"expected (B, H, T, D), got {', '.join(str(tuple(t.shape)) for t in x)}")
    B, _, T, D = q.shape
    if k is not None and (k.shape[0] != B or k.shape[2:] != q.shape[2:] or k.dtype != q.dtype or k.device != q.device):
        raise ValueError(f"q and k differ: {tuple(q.shape)} {q.dtype}, {tuple(k.shape)} {k.dtype}")
    if D not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32/64/128, got {D}")
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"apply_rotary takes bfloat16 or float32 inputs; got {q.dtype}")
    check_tables(cos, sin, D, layout, q.device)
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("the rotary tables take no gradient")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((T,), (B, T)):
            raise ValueError(f"positions must be int32 or int64 ({T},) or ({B}, {T}), got {tuple(positions.shape)} "
                             f"{positions.dtype}")
        if positions.device != q.device:
            raise ValueError(f"positions must be on {q.device}")
        if positions.stride(-1) != 1 and T > 1:
            positions = positions.contiguous()
    _lib.require_gpu(*x)
    if any(t.numel() == 0 for t in x):
        raise ValueError("q and k must not be empty")
    return _Rotary.apply(q, k, cos, sin, positions, layout == "half", False)


__all__ = ["apply_rotary", "ROTARY_LAYOUTS"]
