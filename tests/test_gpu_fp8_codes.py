"""Codes and scales of the quantised rows, bit for bit: scale = max|block| / 448
and code = e4m3(y / scale), each the fp32 division's, as torch computes them on
the CPU from the same values.  (No tolerance: both are single roundings.)"""

import pytest
import torch

from tests.gpu_util import DEV, gen, randn

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def divided(y):
    """(codes as bytes, scales) of rows of fp32 values."""
    assert y.device.type == "cpu" and y.dtype == torch.float32
    rows, cols = y.shape
    wide = torch.nn.functional.pad(y, (0, -cols % 128)).view(rows, -1, 128)
    scales = (wide.abs().amax(-1) / 448.0).clamp_min(2.0 ** -126)
    return (wide / scales[..., None]).to(FP8).view(rows, -1)[:, :cols].contiguous().view(torch.uint8), scales


def same(q, y):
    codes, scales = divided(y)
    assert torch.equal(q.scales.cpu(), scales)
    got = q.values.cpu().contiguous().view(torch.uint8)
    assert torch.equal(got, codes), f"{int((got != codes).sum())} of {codes.numel()} codes"


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(4096, 1024), (333, 1001), (1, 130), (40, 12)], ids=str)
def test_codes_are_those_of_the_division(shape, dtype):
    from logssms_amd.kernel import quantize_fp8
    print(f"codes {shape} {dtype}", flush=True)
    g = gen(shape[0])
    x = (randn(*shape, g=g) * torch.exp(randn(shape[0], 1, g=g))).to(dtype)
    same(quantize_fp8(x.to(DEV)), x.float())


@pytest.mark.parametrize("power", [-146, -140, -126, -117, -90, -81, -80, -72, 0, 60, 118])
def test_codes_at_every_size_of_the_scale(power):
    """Values on the codes' borders and beside them, zeros of both signs, scales
    from the least one to the largest (2^118 * 448 * 1.98 is near the end of fp32)."""
    from logssms_amd.kernel import quantize_fp8
    print(f"codes at 2^{power}", flush=True)
    g = gen(power + 200)
    scale = torch.cat([torch.tensor([1.0, 1.75, 1.5, 2 - 2.0 ** -22, 1 + 2.0 ** -23]), 1 + 0.98 * torch.rand(507, generator=g)])
    # borders: the codes' midpoints, e4m3 with a fourth fraction bit, in its subnormals too
    codes = torch.randint(0, 0x7E, (512, 128), generator=g, dtype=torch.uint8)
    low, high = (c.view(FP8).float() for c in (codes, codes + 1))
    y = (low + high) / 2 * scale[:, None]
    step = torch.randint(-2, 3, (512, 128), generator=g, dtype=torch.int32)
    y = (y.view(torch.int32) + step).view(torch.float32) * torch.where(torch.rand(512, 128, generator=g) < 0.5, -1.0, 1.0)
    y[:, 0] = 448.0 * scale
    y[:, 1], y[:, 2] = 0.0, -0.0
    y = torch.ldexp(y.double(), torch.tensor(power, dtype=torch.float64)).float()
    assert y.isfinite().all()
    same(quantize_fp8(y.to(DEV)), y)


def test_codes_of_the_norms():
    """The norm's own fp32 result is what its rows are quantised from."""
    from logssms_amd.kernel import add_rms_norm_fp8, rms_norm_fp8
    g = gen(6)
    for cols in (200, 1024, 4801, 17000):
        x, res = (randn(64, cols, g=g) for _ in range(2))
        weight = randn(cols, g=g).to(DEV)
        q, y = rms_norm_fp8(x.to(DEV), weight, 1e-6, keep=True)
        same(q, y.cpu())
        q, y, _ = add_rms_norm_fp8(x.to(DEV), res.to(DEV), weight, 1e-6, weight_offset=1.0, keep=True)
        same(q, y.cpu())


@pytest.mark.parametrize("dim", [64, 96])
def test_codes_of_the_gated_norm(dim):
    """Both forms of the gated norm: with a gate of 2^12, silu is the gate itself,
    and a head of equal powers of two has a norm that fp32 holds exactly, so that
    the quantised values are known bit for bit."""
    from logssms_amd.kernel import rms_norm_gated_fp8
    g = gen(dim)
    sign = torch.where(torch.rand(50, 6, dim, generator=g) < 0.5, -1.0, 1.0)
    x = (0.25 * sign).bfloat16()
    gate = torch.full((50, 6, dim), 4096.0).bfloat16()
    weight = randn(dim, g=g, std=0.5)
    got = rms_norm_gated_fp8(x.to(DEV), gate.to(DEV), weight.to(DEV), 0.0)
    # the mean of squares is 2^-4 and its inverse root 4, or the fp32 value beside it
    y = sign * weight * 4096.0
    want = [divided((y * near).reshape(50, -1)) for near in (1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -24)]
    codes = got.values.cpu().contiguous().view(torch.uint8)
    assert any(torch.equal(got.scales.cpu(), s) and torch.equal(codes, c) for c, s in want)


def test_weights_are_quantised_alike_on_every_device():
    from logssms_amd.kernel import quantize_fp8_weight
    w = randn(1000, 1111, g=gen(2)) * torch.exp(randn(1000, 1, g=gen(3)))
    here, there = quantize_fp8_weight(w), quantize_fp8_weight(w.to(DEV))
    assert torch.equal(there.scales.cpu(), here.scales)
    assert torch.equal(there.values.cpu().contiguous().view(torch.uint8), here.values.contiguous().view(torch.uint8))
    # rows of weights and of tokens lie at the same strides
    from logssms_amd.kernel import quantize_fp8
    for cols in (1, 15, 16, 17, 500, 512, 513, 528, 529, 640, 641, 1000, 1024, 1025, 4096):
        x = torch.ones(2, cols)
        assert quantize_fp8(x.to(DEV)).values.stride() == quantize_fp8_weight(x).values.stride(), cols
