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


def _padded(cols: int) -> int:
    return (cols + 15) // 16 * 16


def empty_rows(rows: int, cols: int, device) -> Fp8Tensor:
    """An uninitialised destination of quantised rows.  The scales are laid out
    block by block (strides 1, rows): the product reads one block of many rows
    at a time."""
    values = torch.empty(rows, _padded(cols), dtype=FP8, device=device)
    scales = torch.empty(-(-cols // BLOCK), rows, dtype=torch.float32, device=device)
    return Fp8Tensor(values if values.shape[1] == cols else values[:, :cols], scales.t())


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x`` as [rows, cols] with unit column stride (a copy where it has no such view)."""
    x = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def quantize_fp8(x: torch.Tensor) -> Fp8Tensor:
    """The rows of ``x`` (fp32, bf16 or f16, leading dimensions flattened) in
    8 bits.  A block that holds a NaN or an infinity reads back as NaN."""
    assert x.ndim >= 1 and x.shape[-1] > 0, "rows of at least one value"
    x2 = rows_of(x)
    out = empty_rows(x2.shape[0], x2.shape[1], x2.device)
    _lib.call_on(
        x2, "gdn_quantize_fp8",
        x2.data_ptr(), _lib.dtype_code(x2.dtype), x2.shape[0], x2.shape[1], x2.stride(0), *fp8_args(out),
    )
    return out


def fp8_args(t: Fp8Tensor) -> tuple:
    values, scales = t
    return values.data_ptr(), values.stride(0), scales.data_ptr(), scales.stride(0), scales.stride(1)


def quantize_fp8_weight(weight: torch.Tensor) -> Fp8Tensor:
    """A projection's weights [N, K] with a scale for each 128 x 128 block.
    Once per load: elementary torch operations, on any device."""
    assert weight.ndim == 2 and weight.numel() > 0, "weight must be [N, K]"
    n, k = weight.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, dtype=torch.float32, device=weight.device)
    w[:n, :k] = weight
    w = w.view(nb, BLOCK, kb, BLOCK)
    scales = (w.abs().amax((1, 3)) / _TOP).clamp_min(_LEAST_SCALE)
    w = (w / scales[:, None, :, None]).to(FP8).view(nb * BLOCK, kb * BLOCK)
    # rows at multiples of 16 bytes, zeros behind them
    return Fp8Tensor(w.view(torch.uint8)[:n, :_padded(k)].contiguous().view(FP8)[:, :k], scales)


def _check_values(t: torch.Tensor, name: str) -> None:
    assert t.ndim == 2 and t.dtype == FP8, f"{name} values must be a 2-D float8_e4m3fn tensor"
    rows, cols = t.shape
    assert cols > 0 and (cols == 1 or t.stride(1) == 1), f"{name} values need unit column stride"
    if rows == 0:
        return
    assert t.data_ptr() % 16 == 0 and (rows == 1 or (t.stride(0) % 16 == 0 and t.stride(0) >= cols)), \
        f"the rows of {name} must start at multiples of 16 bytes and not overlap"
    if cols % 16:  # the kernel reads whole 16 bytes
        last = t.storage_offset() + (rows - 1) * t.stride(0) + _padded(cols)
        assert last <= t.untyped_storage().nbytes(), f"the last row of {name} must be readable up to a multiple of 16"


def fp8_linear(x: Fp8Tensor, weight: Fp8Tensor, out_dtype: torch.dtype = torch.bfloat16, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``x [M, K] @ weight [N, K].T`` of quantised operands, accumulated in
    fp32 and rounded once to ``out_dtype`` (bf16 or f16).  ``out`` [M, N] may be
    a view with unit column stride; it is allocated when None."""
    xv, xs = x
    wv, ws = weight
    _check_values(xv, "x")
    _check_values(wv, "weight")
    M, K = xv.shape
    N = wv.shape[0]
    blocks = -(-K // BLOCK)
    assert N > 0 and wv.shape[1] == K, "x [M, K] and weight [N, K] must share K"
    assert xs.dtype == torch.float32 and xs.shape == (M, blocks), "x scales must be fp32 [M, ceil(K / 128)]"
    assert ws.dtype == torch.float32 and ws.shape == (-(-N // BLOCK), blocks), \
        "weight scales must be fp32 [ceil(N / 128), ceil(K / 128)]"
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=xv.device)
    else:
        assert out.shape == (M, N) and out.dtype == out_dtype, "out must be [M, N] of out_dtype"
        assert (N == 1 or out.stride(1) == 1) and (M <= 1 or out.stride(0) >= N), "out needs rows of unit stride"
    assert out_dtype in (torch.bfloat16, torch.float16), "out_dtype must be bfloat16 or float16"
    assert xv.device == xs.device == wv.device == ws.device == out.device, "all operands on one device"
    if M:
        _lib.call_on(
            xv, "gdn_fp8_linear",
            *fp8_args(x), *fp8_args(weight), M, N, K, out.data_ptr(), _lib.dtype_code(out_dtype), out.stride(0),
        )
    return out


__all__ = ["Fp8Tensor", "fp8_linear", "quantize_fp8", "quantize_fp8_weight"]
