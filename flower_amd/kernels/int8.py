"""8-bit rows and the product of int8 matrices, on the HIP library (gfx950).

A row in 8 bits is codes and one float32 scale s = max(max|h| / Q, 1e-12): int8 codes round(h / s) with Q = 127, or
float8_e4m3fn codes of h / s with Q = 448. The passes that make them start from what produces the row, so that a norm's or an
activation's output never goes through memory in 16 bits:

``quant_rows``      the rows as they are
``rms_norm_quant``  RMSNorm (flower/models/base.py:324-338), with the residual's addition before it
``gelu_quant``, ``swiglu_quant``  the MLP's activations (base.py:519-521, :538-550)
``int8_scaled_mm``  the product of int8 rows and int8 weights with a scale for each token and channel
``int8_linear``     ``quant_rows`` and ``int8_scaled_mm``: a linear with int8 weights on 16-bit activations

The reference's 8-bit linears are e4m3 (flower/precision.py); integers run at the same rate on this GPU and are four times
finer near a row's maximum, where a normed activation or a weight has its values. All calls are forward-only
(``flower_amd.int8.Int8Linear`` trains), asynchronous on the current stream, and can be captured in a graph.
"""

from __future__ import annotations

import torch

from .. import _lib


def _e4m3(dtype: torch.dtype) -> bool:
    if dtype not in (torch.int8, torch.float8_e4m3fn):
        raise ValueError(f"codes are int8 or float8_e4m3fn, got {dtype}")
    return dtype == torch.float8_e4m3fn


def quant_rows(x: torch.Tensor, *, dtype: torch.dtype = torch.int8):
    """(codes (.., K), scale (..) float32) of the rows x (.., K), bfloat16 or float32.

    A row that holds a NaN or an infinity cannot be told in int8: its scale is NaN and its codes are 0, so that its products
    are NaN (float8_e4m3fn: a NaN stays one, an infinite row's scale is infinite). K is at most 32768, here and in the calls
    below; rows of any stride are read in place, fastest where they start on 16 bytes and K is a multiple of 8.
    """
    return _lib.native().quant_rows8(x, _e4m3(dtype), _lib.stream_or_none(x))


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: torch.Tensor | None = None,
                   dtype: torch.dtype = torch.int8):
    """(codes, scale) of h = x / sqrt(mean(x^2) + eps) * weight, as ``quant_rows`` gives them; with ``residual`` (as x):
    (codes, scale, sum), where sum = x + residual, rounded to x's type, is what the norm is of.

    weight (K,): float32 or x's type. The norm is in float32 and is rounded once, to its code.
    """
    codes, scale, total = _lib.native().rms_norm_quant(x, weight, eps, residual, _e4m3(dtype), _lib.stream_or_none(x))
    return (codes, scale) if residual is None else (codes, scale, total)


def gelu_quant(x: torch.Tensor, *, dtype: torch.dtype = torch.int8):
    """(codes, scale) of h = x (1 + erf(x / sqrt 2)) / 2, as ``quant_rows`` gives them."""
    return _lib.native().act_quant(x, None, _e4m3(dtype), _lib.stream_or_none(x))


def swiglu_quant(gate: torch.Tensor, up: torch.Tensor, *, dtype: torch.dtype = torch.int8):
    """(codes, scale) of h = gate / (1 + exp(-gate)) * up, as ``quant_rows`` gives them."""
    return _lib.native().act_quant(gate, up, _e4m3(dtype), _lib.stream_or_none(gate))


def int8_scaled_mm(a: torch.Tensor, a_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                   bias: torch.Tensor | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """(.., N) bfloat16: (a . weight^T) a_scale[row] weight_scale[column] + bias, rounded, and added to ``residual``, rounded again.

    a (.., K) and weight (N, K) int8; a_scale float32, one a row or one for all; weight_scale float32, (N,) or one; bias (N,)
    float32 or bfloat16; residual (.., N) bfloat16. The sums are exact (K <= 131071), so the result depends on nothing but
    the inputs: one row gives the same bits alone as in a batch. Any sizes; K % 16 == 0 with 16-byte rows is the fast case.
    """
    return _lib.native().int8_scaled_mm(a, a_scale, weight, weight_scale, bias, residual, _lib.stream_or_none(a))


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *, bias: torch.Tensor | None = None,
                residual: torch.Tensor | None = None) -> torch.Tensor:
    """``int8_scaled_mm`` of the int8 rows (``quant_rows``) of x (.., K), bfloat16 or float32."""
    return _lib.native().int8_linear(x, weight, weight_scale, bias, residual, _lib.stream_or_none(x))


__all__ = ["quant_rows", "rms_norm_quant", "gelu_quant", "swiglu_quant", "int8_scaled_mm", "int8_linear"]
