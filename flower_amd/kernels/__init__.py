"""HIP (gfx950) kernels behind the reference's ``flower.kernels`` operator API."""

from .fp8_swa_attention import (E4M3_MAX, _per_tensor_fp8, amax_e4m3, dequantize_e4m3, fp8_swa_attention,
                                fp8_swa_attention_forward, fp8_swa_attention_from_codes, qk_norm_rope_quant_e4m3,
                                quantize_e4m3_with_amax, reference_swa_attention)
from .int8 import gelu_quant, int8_linear, int8_scaled_mm, quant_rows, rms_norm_quant, swiglu_quant
from .paged import compact_pages, paged_append, paged_attention, reorder_pages, reserve_pages
from .rotary import apply_rotary

__all__ = ["E4M3_MAX", "_per_tensor_fp8", "amax_e4m3", "dequantize_e4m3", "fp8_swa_attention",
           "fp8_swa_attention_forward", "fp8_swa_attention_from_codes", "qk_norm_rope_quant_e4m3",
           "quantize_e4m3_with_amax", "reference_swa_attention",
           "apply_rotary", "paged_append", "paged_attention", "reserve_pages", "reorder_pages", "compact_pages",
           "quant_rows", "rms_norm_quant", "gelu_quant", "swiglu_quant", "int8_scaled_mm", "int8_linear"]
