"""8-bit rows and the int8 linear, restated in numpy. TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

The reference has no integer linears; the definitions are include/flower_amd.h's:
  rows:    scale = max(max|h| / Q, 1e-12) in fp32, code = rne(fp32(h / scale)), Q = 127 (int8) or 448 (e4m3, cast as
           ``oracle.e4m3.f32_to_e4m3``); an int8 row with a value that is not finite: scale NaN, codes 0.
  product: exact integer sums; fp32(sum) * sa * sb (+ bias), rounded to bf16 by the caller.
Pinned by tests/test_oracle_int8.py against torch on the CPU.
"""

from __future__ import annotations

import math

import numpy as np

from .e4m3 import f32_to_e4m3

F32 = np.float32


def rows8(h: np.ndarray, kind: str = "int8"):
    """(codes, scale) of the rows h [R, C], fp32: int8 codes, or e4m3 codes as uint8."""
    h = np.ascontiguousarray(h, dtype=F32)
    amax = np.abs(h).max(axis=1)
    with np.errstate(invalid="ignore", over="ignore"):
        scale = (amax / F32(127.0 if kind == "int8" else 448.0)).astype(F32)
        scale = np.where(scale < F32(1e-12), F32(1e-12), scale)
        units = (h / scale[:, None]).astype(F32)
    if kind == "e4m3":
        return f32_to_e4m3(units), scale
    bad = ~np.isfinite(amax)
    scale[bad] = np.nan
    units[bad] = 0.0
    return np.rint(units).astype(np.int8), scale


def rms_norm(t: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    """In 64 bits."""
    t = t.astype(np.float64)
    return t / np.sqrt((t * t).mean(axis=1, keepdims=True) + eps) * weight.astype(np.float64)


def gelu(x: np.ndarray) -> np.ndarray:
    """In 64 bits."""
    x = x.astype(np.float64)
    return 0.5 * x * np.vectorize(math.erfc)(-x * math.sqrt(0.5)) if x.size else x


def swiglu(gate: np.ndarray, up: np.ndarray) -> np.ndarray:
    """In 64 bits."""
    g = gate.astype(np.float64)
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * up.astype(np.float64)


def product(a: np.ndarray, b: np.ndarray) -> np.ndarray:
    """The integer sums a [M, K] . b [N, K]^T, exact."""
    return (a.astype(np.float64) @ b.astype(np.float64).T).astype(np.int64)
