"""Block-scaled 8-bit projections on the gfx950 kernels (``csrc/fp8_linear.hip``,
``csrc/rms_norm.hip``); the reference has no counterpart.

An ``Fp8Tensor`` holds OCP e4m3 values and fp32 scales: one for each 128
values of a row (activations), or one for each 128 x 128 block (weights).  It
stands for ``value * scale``; ``scale = max|block| / 448``.

    x = quantize_fp8(hidden)                  # or the fp8 norms of kernel.norm
    w = quantize_fp8_weight(linear_weight)    # once, when the weights are loaded
    y = fp8_linear(x, w)                      # bf16 or f16
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib

BLOCK = 128
FP8 = torch.float8_e4m3fn
_TOP = 448.0
_LEAST_SCALE = 2.0 ** -126


class Fp8Tensor(NamedTuple):
    """``values`` [rows, cols] ``float8_e4m3fn`` with unit column stride, rows
    at multiples of 16 bytes and readable up to the next multiple of 16;
    ``scales`` fp32 [rows, ceil(cols / 128)], or [ceil(rows / 128),
    ceil(cols / 128)] for weights, at any strides."""

    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        """The fp32 values it stands for (elementary torch operations)."""
        rows, cols = self.values.shape
        scales = self.scales.repeat_interleave(BLOCK, 1)[:, :cols]
        if self.scales.shape[0] != rows:
            scales = scales.repeat_interleave(BLOCK, 0)[:rows]
        return self.values.float() * scales


def _stride(cols: int) -> int:
    """Of rows in 8 bits: whole cache lines from 513 values on, where that adds at
    most a quarter.  The same rule as ``fp8_stride`` of ``csrc/host.cpp``."""
    return -(-cols // 128) * 128 if cols > 512 else -(-cols // 16) * 16


def quantize_fp8(x: torch.Tensor) -> Fp8Tensor:
    """The rows of ``x`` (fp32, bf16 or f16, leading dimensions flattened) in
    8 bits.  A block that holds a NaN or an infinity reads back as NaN.  The
    scales are laid out block by block (strides 1, rows): the product reads one
    block of many rows at a time."""
    return Fp8Tensor(*_lib.host().quantize_fp8(x))


@torch.no_grad()
def quantize_fp8_weight(weight: torch.Tensor) -> Fp8Tensor:
    """A projection's weights [N, K] with a scale for each 128 x 128 block.
    Once per load: elementary torch operations, on any device, without a gradient."""
    assert weight.ndim == 2 and weight.numel() > 0, "weight must be [N, K]"
    n, k = weight.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, dtype=torch.float32, device=weight.device)
    w[:n, :k] = weight
    w = w.view(nb, BLOCK, kb, BLOCK)
    # by a tensor: on a GPU, torch divides by a number as a product with its reciprocal
    scales = (w.abs().amax((1, 3)) / w.new_tensor(_TOP)).clamp_min(_LEAST_SCALE)
    w = (w / scales[:, None, :, None]).to(FP8).view(nb * BLOCK, kb * BLOCK)
    # rows at multiples of 16 bytes, zeros behind them
    return Fp8Tensor(w.view(torch.uint8)[:n, :_stride(k)].contiguous().view(FP8)[:, :k], scales)


def fp8_linear(x: Fp8Tensor, weight: Fp8Tensor, out_dtype: torch.dtype = torch.bfloat16, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``x [M, K] @ weight [N, K].T`` of quantised operands, accumulated in
    fp32 and rounded once to ``out_dtype`` (bf16 or f16).  ``out`` [M, N] may be
    a view with unit column stride; it is allocated when None."""
    return _lib.host().fp8_linear(x[0], x[1], weight[0], weight[1], out_dtype, out)


__all__ = ["Fp8Tensor", "fp8_linear", "quantize_fp8", "quantize_fp8_weight"]
