"""``RMSNormGated`` (reference ``python/logssms/layers/norm.py:42-53``): the
output norm ``GatedDeltaNet.output`` applies to the core output
(``python/logssms/layers/gated_delta.py:133-139``); and ``RMSNorm``, the norm in
front of a layer with the residual's addition."""

from __future__ import annotations

import torch

from ..kernel.fp8 import Fp8Tensor
from ..kernel.norm import (add_rms_norm, add_rms_norm_fp8, rms_norm, rms_norm_fp8, rms_norm_gated,
                           rms_norm_gated_fp8)


class RMSNorm:
    """``weight_offset`` 1 for models that store the weight's distance from one."""

    def __init__(self, size: int, eps: float, weight_offset: float = 0.0) -> None:
        self.eps = eps
        self.weight_offset = weight_offset
        self.weight = torch.full((size,), 1.0 - weight_offset, dtype=torch.float32)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """The norm of ``x``, or of ``x + residual`` with the sum, the next residual."""
        if residual is None:
            return rms_norm(x, self.weight, self.eps, weight_offset=self.weight_offset)
        return add_rms_norm(x, residual, self.weight, self.eps, weight_offset=self.weight_offset)

    def forward_fp8(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """``forward`` with its result in 8 bits in front: what a layer with
        8-bit projections takes beside ``x``."""
        if residual is None:
            return rms_norm_fp8(x, self.weight, self.eps, weight_offset=self.weight_offset, keep=True)
        return add_rms_norm_fp8(x, residual, self.weight, self.eps, weight_offset=self.weight_offset, keep=True)


class RMSNormGated:
    def __init__(self, size: int, eps: float) -> None:
        self.eps = eps
        self.weight = torch.ones(size, dtype=torch.float32)

    def forward(self, hidden_states: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        return rms_norm_gated(hidden_states, gate, self.weight, self.eps)

    def forward_fp8(self, hidden_states: torch.Tensor, gate: torch.Tensor) -> Fp8Tensor:
        """[tokens, heads, dim] -> the rows of heads * dim values in 8 bits."""
        return rms_norm_gated_fp8(hidden_states, gate, self.weight, self.eps)


__all__ = ["RMSNorm", "RMSNormGated"]
