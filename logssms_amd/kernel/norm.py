"""``rms_norm_gated`` (drop-in for the reference's ``python/logssms/kernel/norm.py:151-187``),
on the gfx950 kernel ``gdn_rms_norm_gated`` (``csrc/norm.hip``), and the norms
either side of a layer with 8-bit projections (``csrc/rms_norm.hip``; no
counterpart in the reference): ``rms_norm`` and ``add_rms_norm`` with outputs in
the io type, ``rms_norm_fp8``, ``add_rms_norm_fp8`` and ``rms_norm_gated_fp8``
with quantised rows (``kernel.fp8.Fp8Tensor``)."""

from __future__ import annotations

import torch

from .. import _lib
from .fp8 import Fp8Tensor, empty_rows, fp8_args, rows_of


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


def _norm(x, residual, weight, eps, weight_offset, residual_out, quantize, keep):
    cols = x.shape[-1]
    assert x.ndim >= 1 and cols > 0 and weight.shape == (cols,), "weight must be [x.shape[-1]]"
    assert weight.device == x.device, "all operands on one device"
    x2 = rows_of(x)
    weight = weight.contiguous()
    res2 = sum2 = None
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype and residual.device == x.device, \
            "the residual must be like x"
        res2 = rows_of(residual)
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        assert residual_out.shape == x.shape and residual_out.dtype == x.dtype and residual_out.device == x.device, \
            "residual_out must be like x"
        sum2 = residual_out.view(-1, cols)
        assert (cols == 1 or sum2.stride(1) == 1) and (sum2.shape[0] <= 1 or sum2.stride(0) >= cols), \
            "residual_out needs rows of unit stride"
    rows = x2.shape[0]
    q = empty_rows(rows, cols, x.device) if quantize else None
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if keep else None
    _lib.call_on(
        x2, "gdn_rms_norm",
        x2.data_ptr(), _lib.dtype_code(x2.dtype), rows, cols, x2.stride(0),
        _lib.ptr(res2), 0 if res2 is None else res2.stride(0), weight.data_ptr(), _lib.dtype_code(weight.dtype),
        float(weight_offset), float(eps), _lib.ptr(sum2), 0 if sum2 is None else sum2.stride(0), _lib.ptr(y), cols,
        *(fp8_args(q) if quantize else (None, 0, None, 0, 0)),
    )
    return q, y, residual_out


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, *, weight_offset: float = 0.0) -> torch.Tensor:
    """Per row of ``x.shape[-1]`` channels: ``x * rsqrt(mean(x^2) + eps) *
    (weight + weight_offset)``, computed in fp32, in the dtype and shape of ``x``
    (``weight_offset`` 1 for models that store the weight's distance from one)."""
    return _norm(x, None, weight, eps, weight_offset, None, False, True)[1]


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                 weight_offset: float = 0.0, residual_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """``rms_norm(x + residual)`` and the sum itself, the next residual, rounded
    to the dtype of ``x`` (the norm takes the unrounded sum).  ``residual_out``
    may be ``residual``, which is then updated in place; it is allocated when None."""
    _, y, total = _norm(x, residual, weight, eps, weight_offset, residual_out, False, True)
    return y, total


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float, *, weight_offset: float = 0.0,
                 keep: bool = False) -> Fp8Tensor | tuple[Fp8Tensor, torch.Tensor]:
    """``rms_norm`` in 8 bits (leading dimensions flattened), quantised from the
    fp32 result; with ``keep`` also the result in the dtype of ``x``."""
    q, y, _ = _norm(x, None, weight, eps, weight_offset, None, True, keep)
    return (q, y) if keep else q


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                     weight_offset: float = 0.0, keep: bool = False, residual_out: torch.Tensor | None = None
                     ) -> tuple[Fp8Tensor, torch.Tensor] | tuple[Fp8Tensor, torch.Tensor, torch.Tensor]:
    """``add_rms_norm`` in 8 bits: the quantised rows, with ``keep`` the result
    in the dtype of ``x``, and the sum."""
    q, y, total = _norm(x, residual, weight, eps, weight_offset, residual_out, True, keep)
    return (q, y, total) if keep else (q, total)


def rms_norm_gated_fp8(hidden_states: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, eps: float
                       ) -> Fp8Tensor:
    """``rms_norm_gated`` of [tokens, heads, dim], quantised over each token's
    flattened row of ``heads * dim`` values."""
    assert hidden_states.ndim == 3 and hidden_states.shape == gate.shape, "[tokens, heads, dim] expected"
    assert hidden_states.dtype == gate.dtype, "hidden states and gate of one dtype"
    assert hidden_states.device == gate.device == weight.device, "all operands on one device"
    tokens, heads, dim = hidden_states.shape
    assert heads > 0 and weight.shape == (dim,), "weight must be [dim]"
    hidden, gate = (t if t.stride(2) == 1 or dim == 1 else t.contiguous() for t in (hidden_states, gate))
    weight = weight.contiguous()
    out = empty_rows(tokens, heads * dim, hidden.device)
    _lib.call_on(
        hidden, "gdn_rms_norm_gated_fp8",
        hidden.data_ptr(), _lib.dtype_code(hidden.dtype), tokens, heads, dim, hidden.stride(0), hidden.stride(1),
        gate.data_ptr(), gate.stride(0), gate.stride(1), weight.data_ptr(), _lib.dtype_code(weight.dtype), float(eps),
        *fp8_args(out),
    )
    return out


__all__ = ["add_rms_norm", "add_rms_norm_fp8", "rms_norm", "rms_norm_fp8", "rms_norm_gated", "rms_norm_gated_fp8"]
