"""Kernel entry points mirroring ``logssms.kernel`` for the GDN path."""

from .fp8 import Fp8Tensor, fp8_linear, quantize_fp8, quantize_fp8_weight
from .fused import prepare_gdn
from .norm import add_rms_norm, add_rms_norm_fp8, rms_norm, rms_norm_fp8, rms_norm_gated, rms_norm_gated_fp8
from .paged_attention import append_paged_kv, paged_attention
from .rotary import Rotary, apply_rotary, rotary_embedding
from .store import store_state

__all__ = ["Fp8Tensor", "Rotary", "add_rms_norm", "add_rms_norm_fp8", "append_paged_kv", "apply_rotary", "fp8_linear",
           "paged_attention", "prepare_gdn", "quantize_fp8", "quantize_fp8_weight", "rms_norm", "rms_norm_fp8",
           "rms_norm_gated", "rms_norm_gated_fp8", "rotary_embedding", "store_state"]
