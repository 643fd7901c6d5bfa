"""Block-scaled 8-bit values, the norms that write them and the product that
reads them, in float64 torch from their definitions (no counterpart in the
reference).  ``q`` stands for ``value * scale`` with one scale for each 128
values of a row, or for each 128 x 128 block of weights."""

import torch

BLOCK = 128
TOP = 448.0
LEAST_SCALE = 2.0 ** -126
HALF_STEP = 2.0 ** -4  # e4m3: three fraction bits, half a step relative to the value
HALF_STEP_SUBNORMAL = 2.0 ** -10  # values below 2^-6 lie 2^-9 apart


def block_scales(y):
    """The scales of the rows of ``y`` [rows, cols]."""
    return torch.stack([p.abs().amax(1) for p in y.double().split(BLOCK, 1)], 1).div(TOP).clamp_min(LEAST_SCALE)


def spread(scales, rows, cols):
    """Row or block scales as one per value."""
    out = scales.double().repeat_interleave(BLOCK, 1)[:, :cols]
    return out if scales.shape[0] == rows else out.repeat_interleave(BLOCK, 0)[:rows]


def dequantize(values, scales):
    return values.double() * spread(scales, *values.shape)


def rms_norm(x, weight, eps, residual=None, weight_offset=0.0):
    """(h, y) of h = x + residual, y = h / sqrt(mean(h^2) + eps) * (weight + offset)."""
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.double() + weight_offset)


def rms_norm_gated(x, gate, weight, eps):
    """[tokens, heads, dim] -> the gated norm, rows flattened."""
    z = gate.double()
    _, y = rms_norm(x, weight, eps)
    return (y * z * torch.sigmoid(z)).flatten(1)


def linear(x, x_scales, weight, weight_scales):
    return dequantize(x, x_scales) @ dequantize(weight, weight_scales).t()


def linear_bound(x, x_scales, weight, weight_scales):
    """How far fp32 sums of the 8-bit matrix instructions may lie from
    ``linear``.  Of each eight consecutive products the instruction keeps what
    lies at least 2^-13 of the largest one's power of two (the power of two of
    a product of two significands in [1, 2) may be one above either's): the
    other seven lose less than 2^-12 of the largest each.  The groups of a
    block, and then the blocks, are added in fp32: K / 8 + K / 128 + 2 additions
    and roundings of at most 2^-23 of the sum of magnitudes."""
    a, b = dequantize(x, x_scales).abs(), dequantize(weight, weight_scales).abs()
    k = a.shape[1]
    pad = (-k) % 8
    a, b = (torch.nn.functional.pad(t, (0, pad)) for t in (a, b))
    largest = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device=a.device)
    total = torch.zeros_like(largest)
    for g in range(0, k, 8):
        products = a[:, None, g:g + 8] * b[None, :, g:g + 8]
        largest += products.amax(-1)
        total += products.sum(-1)
    return 7 * 2.0 ** -12 * largest + (k / 8 + k / 128 + 2) * 2.0 ** -23 * total
