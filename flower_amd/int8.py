"""Linears in 8-bit integers: int8 weights with a scale a channel, int8 activations with a scale a token.

``Int8Linear``            an ``nn.Linear`` whose forward is ``flower_amd.kernels.int8_linear``. Trainable, straight through
                          the quantisers: the gradient products are the e4m3 ones of the "rowwise" recipe
                          (``flower_amd.precision``), whose range a gradient's rows need; ``backward_fp8 = False`` takes bf16.
``int8_linear_train``     its forward as a function, differentiable in input, weight, bias and residual
``convert_model_to_int8`` replaces a model's linears as ``convert_model_to_fp8`` does (flower/precision.py:134-195), by the
                          same rules; ``fp8_weight_cache`` then keeps the int8 codes for the length of its block.

Rows in 8 bits hold at most 32768 values (``flower_amd.kernels.quant_rows``): so many input features, and any number of outputs.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from .kernels.int8 import int8_scaled_mm, quant_rows
from .precision import Fp8Linear, fp8_module_filter, quantize_weight_cols

MAX_IN_FEATURES = 32768


def _row_type(t: torch.Tensor | None) -> torch.Tensor | None:
    """t in a type that the operators take: bfloat16 unless it is that or float32."""
    return t if t is None or t.dtype in (torch.bfloat16, torch.float32) else t.to(torch.bfloat16)


def quantize_weight_int8(weight: torch.Tensor):
    """(codes (N, K) int8, scale (N,) float32) of a weight: one scale an output channel."""
    return quant_rows(_row_type(weight.detach()))


def int8_linear_train(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                      residual: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight^T + bias``, plus ``residual``, in int8: both operands quantised now, a scale a token and a channel; bf16 out.
    x (.., K), K <= 32768, weight (N, K) and bias (N,) bf16 or fp32, residual bf16; for a gradient at most 65535 * 256 fp32 rows.
    Differentiable once by backward, as ``Int8Linear`` is."""
    return _lib.native().int8_linear_train(x, weight, bias, residual, None, None, None, None, True, _lib.stream_or_none(x))


def _check_width(in_features: int) -> None:
    if in_features > MAX_IN_FEATURES:
        raise ValueError(f"an Int8Linear takes at most {MAX_IN_FEATURES} input features, got {in_features}")


class Int8Linear(Fp8Linear):
    """``nn.Linear`` in int8 (see the module). Shares the Parameters of the Linear it was built from. The weight is quantised
    on every call unless an ``fp8_weight_cache`` is active. At most 32768 input features. ``forward_codes`` takes the input as
    codes and scales already, from ``rms_norm_quant`` or another of the passes of ``flower_amd.kernels``. The output is bfloat16;
    inputs and Parameters that are neither bfloat16 nor float32 are cast to it."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None) -> None:
        _check_width(in_features)
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.recipe = "int8"

    @classmethod
    def from_linear(cls, lin: nn.Linear) -> "Int8Linear":
        _check_width(lin.in_features)
        new = super().from_linear(lin)
        new.recipe = "int8"
        return new

    def quantize_weight(self):
        return quantize_weight_int8(self.weight)

    def tensorwise_codes(self):
        raise RuntimeError("an Int8Linear has no tensorwise codes")

    def weight_col_codes(self):
        cached = getattr(self, "_fp8_cached_cols", None)
        if cached is not None:
            return cached
        codes = quantize_weight_cols(self.weight, "rowwise")
        self._keep_cols(codes)
        return codes

    def forward_with(self, x: torch.Tensor, w8: torch.Tensor, w_scale: torch.Tensor, x_amax=None, residual=None,
                     w8t=None) -> torch.Tensor:
        """x_amax and w8t are of the tensorwise recipe: not used."""
        if torch.is_autocast_enabled("cuda"):
            x = x.to(torch.get_autocast_dtype("cuda"))
        x = _row_type(x)
        cols = (None, None)
        if (getattr(self, "_fp8_cached", None) is not None and self.backward_fp8 and torch.is_grad_enabled() and x.requires_grad
                and self.in_features % 16 == 0 and self.out_features % 16 == 0):
            cols = self.weight_col_codes()              # kept for the cache's length; without one the backward makes its own
        return _lib.native().int8_linear_train(x, _row_type(self.weight), _row_type(self.bias), residual, w8, w_scale, *cols,
                                               self.backward_fp8, _lib.stream_or_none(x))

    def forward(self, x: torch.Tensor, x_amax=None, residual=None) -> torch.Tensor:
        return self.forward_with(x, *self.weight_codes(), residual=residual)

    @torch.no_grad()
    def forward_codes(self, codes: torch.Tensor, scale: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """The output for an input in int8: codes (.., in_features) and scale (..). Forward-only."""
        return int8_scaled_mm(codes, scale, *self.weight_codes(), bias=_row_type(self.bias), residual=residual)


def convert_model_to_int8(model: nn.Module, *, keep_bf16_blocks: int = 1, verbose: bool = True):
    """Replace every Linear that ``fp8_module_filter`` admits, of at most 32768 input features, by an ``Int8Linear`` sharing its
    Parameters, in place; returns (model, info). As ``convert_model_to_fp8``, it refuses a model without ``blocks``."""
    num_layers = len(getattr(model, "blocks", []))
    if num_layers == 0:
        raise RuntimeError("convert_model_to_int8 found no `blocks` on the model; the block-range guardrail cannot be applied. "
                           "Refusing to convert blindly.")
    admit = fp8_module_filter(num_layers, keep_bf16_blocks)
    named = list(model.named_modules())
    targets = [(fqn, m) for fqn, m in named if admit(m, fqn) and m.in_features <= MAX_IN_FEATURES]
    for fqn, mod in targets:
        owner, _, attr = fqn.rpartition(".")
        setattr(model.get_submodule(owner) if owner else model, attr, Int8Linear.from_linear(mod))
    info = {"int8_keep_bf16_blocks": keep_bf16_blocks, "int8_converted_linears": len(targets),
            "int8_total_linears": sum(isinstance(m, nn.Linear) for _, m in named)}
    if verbose:
        print(f"[int8] converted {len(targets)}/{info['int8_total_linears']} Linear layers (blocks {keep_bf16_blocks}.."
              f"{num_layers - keep_bf16_blocks - 1} of {num_layers}; first/last {keep_bf16_blocks} stay as they are)", flush=True)
    return model, info


__all__ = ["Int8Linear", "int8_linear_train", "convert_model_to_int8", "quantize_weight_int8"]
