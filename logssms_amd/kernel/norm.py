"""``rms_norm_gated`` (drop-in for the reference's ``python/logssms/kernel/norm.py:151-187``),
on the gfx950 kernel ``gdn_rms_norm_gated`` (``csrc/norm.hip``), and the norms
either side of a layer with 8-bit projections (``csrc/rms_norm.hip``; no
counterpart in the reference): ``rms_norm`` and ``add_rms_norm`` with outputs in
the io type, ``rms_norm_fp8``, ``add_rms_norm_fp8`` and ``rms_norm_gated_fp8``
with quantised rows (``kernel.fp8.Fp8Tensor``)."""

from __future__ import annotations

import torch

from .. import _lib
from .fp8 import Fp8Tensor


def rms_norm_gated(
    hidden_states: torch.Tensor,
    gate: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
) -> torch.Tensor:
    """Per row of ``hidden_states.shape[-1]`` channels:
    ``(x * rsqrt(mean(x^2) + eps)) * weight * silu(gate)``, computed in fp32 and
    returned in the dtype and shape of ``hidden_states``.  ``gate`` may be a
    strided view (the reference indexes it as ``gate.reshape(-1, gate.shape[-2], n)``)."""
    assert hidden_states.shape == gate.shape
    assert hidden_states.shape[-1] == weight.numel()
    assert hidden_states.is_cuda and gate.is_cuda and weight.is_cuda
    num_cols = hidden_states.shape[-1]
    hidden = hidden_states.reshape(-1, num_cols).contiguous()
    gate3 = gate.reshape(-1, gate.shape[-2], num_cols) if gate.ndim > 1 else gate.view(1, 1, num_cols)
    weight = weight.contiguous()
    output = torch.empty_like(hidden)
    _lib.call(
        "gdn_rms_norm_gated",
        hidden.data_ptr(), _lib.dtype_code(hidden.dtype), hidden.shape[0], num_cols,
        gate3.data_ptr(), _lib.dtype_code(gate3.dtype), gate3.shape[1], gate3.stride(0), gate3.stride(1),
        gate3.stride(2), weight.data_ptr(), _lib.dtype_code(weight.dtype), float(eps), output.data_ptr(),
        _lib.stream_of(hidden),
    )
    return output.view(hidden_states.shape)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, *, weight_offset: float = 0.0) -> torch.Tensor:
    """Per row of ``x.shape[-1]`` channels: ``x * rsqrt(mean(x^2) + eps) *
    (weight + weight_offset)``, computed in fp32, in the dtype and shape of ``x``
    (``weight_offset`` 1 for models that store the weight's distance from one)."""
    return _lib.host().rms_norm(x, None, weight, eps, weight_offset, None, False, True)[2]


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                 weight_offset: float = 0.0, residual_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """``rms_norm(x + residual)`` and the sum itself, the next residual, rounded
    to the dtype of ``x`` (the norm takes the unrounded sum).  ``residual_out``
    may be ``residual`` or ``x``, which is then updated in place; it is allocated when None."""
    _, _, y, total = _lib.host().rms_norm(x, residual, weight, eps, weight_offset, residual_out, False, True)
    return y, total


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float, *, weight_offset: float = 0.0,
                 keep: bool = False) -> Fp8Tensor | tuple[Fp8Tensor, torch.Tensor]:
    """``rms_norm`` in 8 bits (leading dimensions flattened), quantised from the
    fp32 result; with ``keep`` also the result in the dtype of ``x``."""
    values, scales, y, _ = _lib.host().rms_norm(x, None, weight, eps, weight_offset, None, True, keep)
    q = Fp8Tensor(values, scales)
    return (q, y) if keep else q


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                     weight_offset: float = 0.0, keep: bool = False, residual_out: torch.Tensor | None = None
                     ) -> tuple[Fp8Tensor, torch.Tensor] | tuple[Fp8Tensor, torch.Tensor, torch.Tensor]:
    """``add_rms_norm`` in 8 bits: the quantised rows, with ``keep`` the result
    in the dtype of ``x``, and the sum."""
    values, scales, y, total = _lib.host().rms_norm(x, residual, weight, eps, weight_offset, residual_out, True, keep)
    q = Fp8Tensor(values, scales)
    return (q, y, total) if keep else (q, total)


def rms_norm_gated_fp8(hidden_states: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, eps: float
                       ) -> Fp8Tensor:
    """``rms_norm_gated`` of [tokens, heads, dim], quantised over each token's
    flattened row of ``heads * dim`` values."""
    return Fp8Tensor(*_lib.host().rms_norm_gated_fp8(hidden_states, gate, weight, eps))


__all__ = ["add_rms_norm", "add_rms_norm_fp8", "rms_norm", "rms_norm_fp8", "rms_norm_gated", "rms_norm_gated_fp8"]
