"""Run-time resource contract of the fused prefill path (mirror of the reference's
``src/mega_attention/runtime/__init__.py:1-3``), plus the per-layer serving wrapper the
reference only sketches in its design notes."""
from .workspace import FusedFaOprojArWorkspace
from .prefill_layer import FusedPrefillLayer

from .residual_rmsnorm import residual_rmsnorm
from .rope import rope_qk_
from .rmsnorm_int8 import residual_rmsnorm_int8, rmsnorm_int8
from .linear_int8 import check_linear_status, dequantize_int8, linear_int8, quantize_weight_int8
from .rope_append import rope_append

__all__ = ["FusedFaOprojArWorkspace", "FusedPrefillLayer", "residual_rmsnorm", "rope_qk_", "rmsnorm_int8",
           "residual_rmsnorm_int8", "linear_int8", "quantize_weight_int8", "dequantize_int8",
           "check_linear_status", "rope_append"]
