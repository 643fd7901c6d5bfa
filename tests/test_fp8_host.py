"""Block-scaled 8-bit operators on the CPU: the oracle against torch's own
float8 conversion and products, weight quantisation, and every refusal that is
made before a launch."""

import os

import pytest
import torch

from oracle import fp8 as ref

FP8 = torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _built():
    from logssms_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.lib()


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 131), (300, 257), (5, 1000)])
def test_weight_quantisation_rounds_by_half_a_step(n, k):
    from logssms_amd.kernel.fp8 import quantize_fp8_weight
    w = torch.randn(n, k, generator=_gen(n + k)) * torch.exp(2 * torch.randn(n, 1, generator=_gen(1)))
    w[:, k // 2] = 0
    q = quantize_fp8_weight(w)
    assert q.values.shape == (n, k) and q.values.dtype == FP8 and q.values.stride(1) == 1
    assert n == 1 or q.values.stride(0) % 16 == 0
    assert q.scales.shape == (-(-n // 128), -(-k // 128))
    s = ref.spread(q.scales, n, k)
    err = (ref.dequantize(q.values, q.scales) - w.double()).abs()
    # half a step of the code, and 2^-23 for the fp32 division in front of it
    assert (err <= w.double().abs() * (ref.HALF_STEP + 2.0 ** -23) + s * ref.HALF_STEP_SUBNORMAL).all()
    for i in range(q.scales.shape[0]):
        for j in range(q.scales.shape[1]):
            block = w[128 * i:128 * i + 128, 128 * j:128 * j + 128]
            want = max(float(block.abs().max()) / 448, 2.0 ** -126)
            assert abs(float(q.scales[i, j]) - want) <= want * 2.0 ** -23
    assert torch.equal(q.dequantize(), ref.dequantize(q.values, q.scales).float())


def test_weight_quantisation_of_zeros_and_of_what_is_not_finite():
    from logssms_amd.kernel.fp8 import quantize_fp8_weight
    w = torch.zeros(256, 256)
    w[0, 0], w[130, 3], w[140, 200] = float("nan"), float("inf"), -2.0
    q = quantize_fp8_weight(w)
    d = ref.dequantize(q.values, q.scales)
    assert d[:128, :128].isnan().all() and d[128:, :128].isnan().all()
    assert (d[:128, 128:] == 0).all() and float(d[140, 200]) == pytest.approx(-2.0, rel=2.0 ** -22)
    assert float(q.scales[0, 1]) == 2.0 ** -126


def test_oracle_product_and_norms_against_torch():
    g = _gen(3)
    x, w = torch.randn(5, 300, generator=g), torch.randn(140, 300, generator=g)
    xs = ref.block_scales(x)
    xq = (x / ref.spread(xs, 5, 300)).to(FP8)
    ws = torch.rand(2, 3, generator=g) + 0.5
    wq = w.to(FP8)
    got = ref.linear(xq, xs, wq, ws)
    want = torch.zeros(5, 140, dtype=torch.float64)
    for n in range(140):
        for b in range(3):
            part = slice(128 * b, min(300, 128 * b + 128))
            want[:, n] += (xq[:, part].double() @ wq[n, part].double()) * xs[:, b] * float(ws[n // 128, b])
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)
    assert (ref.linear_bound(xq, xs, wq, ws) < 1e-2 * (xq.double().abs() @ wq.double().abs().t())).all()
    weight = torch.rand(300, generator=g)
    h, y = ref.rms_norm(x, weight, 1e-6, residual=x, weight_offset=1.0)
    torch.testing.assert_close(y, torch.nn.functional.rms_norm(2 * x.double(), (300,), weight.double() + 1, 1e-6))
    gate = torch.randn(5, 3, 100, generator=g)
    want = torch.nn.functional.rms_norm(x.view(5, 3, 100).double(), (100,), weight[:100].double(), 1e-6)
    torch.testing.assert_close(ref.rms_norm_gated(x.view(5, 3, 100), gate, weight[:100], 1e-6),
                               (want * torch.nn.functional.silu(gate.double())).flatten(1))


def _pair(rows, cols, scale_rows=None):
    from logssms_amd.kernel import Fp8Tensor
    wide = (cols + 15) // 16 * 16
    return Fp8Tensor(torch.zeros(rows, wide).to(FP8)[:, :cols],
                     torch.ones(rows if scale_rows is None else scale_rows, -(-cols // 128)))


def test_fp8_linear_refuses_what_does_not_fit():
    """Operands that do not fit each other or the kernel, before anything is launched."""
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    _built()
    x, w = _pair(3, 256), _pair(200, 256, 2)
    bad = [
        (_pair(3, 128), w),  # another K
        (Fp8Tensor(x.values.float(), x.scales), w),  # not 8 bits
        (Fp8Tensor(x.values[0], x.scales), w),  # one dimension
        (Fp8Tensor(x.values, x.scales[:, :1]), w),  # a block's scales missing
        (Fp8Tensor(x.values, x.scales[:2]), w),
        (Fp8Tensor(x.values, x.scales.double()), w),
        (x, Fp8Tensor(w.values, w.scales[:1])),
        (x, Fp8Tensor(w.values, torch.ones(200, 2))),  # per-row weight scales
        (Fp8Tensor(torch.zeros(256, 3).to(FP8).t(), x.scales), w),  # K is not the unit stride
        (Fp8Tensor(torch.zeros(3, 264).to(FP8)[:, 8:], x.scales), w),  # rows off 16 bytes
        (Fp8Tensor(torch.zeros(1, 256).to(FP8).expand(3, 256), x.scales), w),  # rows on top of each other
        (Fp8Tensor(torch.zeros(3, 250).to(FP8), torch.ones(3, 2)), Fp8Tensor(torch.zeros(4, 256).to(FP8)[:, :250],
                                                                             torch.ones(1, 2))),
        # the last row ends in the middle of 16 bytes, and so does its storage
        (Fp8Tensor(torch.zeros(250).to(FP8).view(1, 250), torch.ones(1, 2)),
         Fp8Tensor(torch.zeros(4, 256).to(FP8)[:, :250], torch.ones(1, 2))),
    ]
    for a, b in bad:
        with pytest.raises(AssertionError):
            fp8_linear(a, b)
    with pytest.raises(AssertionError):
        fp8_linear(x, w, torch.float32)
    for out in (torch.empty(3, 199, dtype=torch.bfloat16), torch.empty(3, 200), torch.empty(200, 3).bfloat16().t(),
                torch.empty(1, 200, dtype=torch.bfloat16).expand(3, 200)):
        with pytest.raises(AssertionError):
            fp8_linear(x, w, out=out)
    with pytest.raises(RuntimeError, match="ROCm"):
        fp8_linear(x, w)
    assert fp8_linear(_pair(0, 256), w).shape == (0, 200)  # nothing to do


def test_row_operators_refuse_what_does_not_fit():
    from logssms_amd.kernel import (add_rms_norm, add_rms_norm_fp8, quantize_fp8, rms_norm, rms_norm_fp8,
                                    rms_norm_gated_fp8)
    _built()
    x, w = torch.zeros(4, 64), torch.ones(64)
    for call in (
        lambda: rms_norm(x, torch.ones(63), 1e-6),
        lambda: rms_norm(x, torch.ones(1, 64), 1e-6),
        lambda: add_rms_norm(x, x[:3], w, 1e-6),
        lambda: add_rms_norm(x, x.half(), w, 1e-6),
        lambda: add_rms_norm_fp8(x, x, w, 1e-6, residual_out=torch.zeros(4, 63)),
        lambda: add_rms_norm_fp8(x, x, w, 1e-6, residual_out=torch.zeros(64, 4).t()),
        lambda: add_rms_norm_fp8(x, x, w, 1e-6, residual_out=torch.zeros(1, 64).expand(4, 64)),
        lambda: rms_norm_fp8(torch.zeros(4, 0), torch.ones(0), 1e-6),
        lambda: quantize_fp8(torch.zeros(4, 0)),
        lambda: quantize_fp8(torch.zeros(())),
        lambda: rms_norm_gated_fp8(x.view(4, 2, 32), x.view(4, 2, 32).half(), torch.ones(32), 1e-6),
        lambda: rms_norm_gated_fp8(x.view(4, 2, 32), x.view(4, 2, 32), torch.ones(64), 1e-6),
        lambda: rms_norm_gated_fp8(x, x, w, 1e-6),
    ):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: rms_norm(x, w, 1e-6), lambda: quantize_fp8(x),
                 lambda: rms_norm_gated_fp8(x.view(4, 2, 32), x.view(4, 2, 32), torch.ones(32), 1e-6)):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()
    with pytest.raises(TypeError):
        quantize_fp8(torch.zeros(4, 64, dtype=torch.int32))


def test_entry_points_check_before_they_launch():
    """Without a GPU a launch would come back as GDN_ERR_HIP (3); the dummy
    16-byte aligned address is never dereferenced."""
    lib = _built()
    d = 0x10000

    def norm(rows=4, cols=64, dtype=1, x=d, res=None, weight=d, wdt=0, res_out=None, out=d, values=None, vs=64,
             scales=None):
        return lib.gdn_rms_norm(x, dtype, rows, cols, cols, res, cols, weight, wdt, 0.0, 1e-6, res_out, cols, out, cols,
                                values, vs, scales, 1, 4, None)

    assert norm(rows=0, x=None, out=None) == 0
    for kw in (dict(rows=-1), dict(cols=0), dict(dtype=3), dict(wdt=-1), dict(x=None), dict(weight=None),
               dict(out=None), dict(res_out=d), dict(values=d), dict(scales=d), dict(values=d + 8, scales=d),
               dict(values=d, scales=d, vs=72), dict(values=d, scales=d, vs=48), dict(values=d, scales=d + 2),
               dict(rows=1 << 40)):
        assert norm(**kw) == 1, kw
        assert b"gdn_rms_norm:" in lib.gdn_last_error()

    def quantize(rows=4, cols=64, dtype=1, x=d, values=d, vs=64, scales=d):
        return lib.gdn_quantize_fp8(x, dtype, rows, cols, cols, values, vs, scales, 1, 4, None)

    assert quantize(rows=0, x=None) == 0
    for kw in (dict(rows=-1), dict(cols=0), dict(dtype=9), dict(x=None), dict(values=None), dict(scales=None),
               dict(vs=60), dict(rows=1 << 31)):
        assert quantize(**kw) == 1, kw
        assert b"gdn_quantize_fp8:" in lib.gdn_last_error()

    def gated(tokens=4, heads=2, dim=64, dtype=1, x=d, gate=d, weight=d, values=d, vs=128, scales=d):
        return lib.gdn_rms_norm_gated_fp8(x, dtype, tokens, heads, dim, 128, 64, gate, 128, 64, weight, 0, 1e-6, values,
                                          vs, scales, 1, 4, None)

    assert gated(tokens=0, x=None) == 0
    for kw in (dict(tokens=-1), dict(heads=0), dict(dim=0), dict(dtype=9), dict(x=None), dict(gate=None),
               dict(weight=None), dict(values=None), dict(vs=112), dict(heads=1 << 20, dim=1 << 20)):
        assert gated(**kw) == 1, kw
        assert b"gdn_rms_norm_gated_fp8:" in lib.gdn_last_error()
    assert gated(heads=16385, vs=16385 * 64) == 2

    def linear(M=4, N=64, K=128, x=d, xst=128, xs=d, xsr=1, w=d, wst=128, ws=d, out=d, odt=1, ost=64):
        return lib.gdn_fp8_linear(x, xst, xs, xsr, 4, w, wst, ws, 1, 1, M, N, K, out, odt, ost, None)

    assert linear(M=0, x=None, out=None) == 0
    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(odt=0), dict(x=None), dict(xs=None), dict(w=None), dict(ws=None),
               dict(out=None), dict(xst=120), dict(xst=112), dict(wst=136), dict(x=d + 8), dict(w=d + 1), dict(ost=63),
               dict(out=d + 1), dict(xsr=-1)):
        assert linear(**kw) == 1, kw
        assert b"gdn_fp8_linear:" in lib.gdn_last_error()
    for kw in (dict(xst=1 << 24), dict(wst=1 << 24), dict(xsr=1 << 22)):
        assert linear(**kw) == 2, kw


def test_norm_counts_the_threads_of_a_row():
    """A launch holds fewer than 2^32 threads; a row of up to 128 values takes
    16 of them, one of up to 6144 768, a wider one all 1024 of a block."""
    lib = _built()
    d = 0x10000
    for rows, cols in ((1 << 22, 6152), (1 << 22, 8192), (6 << 20, 4104), (1 << 23, 4096), (1 << 25, 1000), (1 << 28, 64),
                       (1 << 62, 8)):
        rc = lib.gdn_rms_norm(d, 1, rows, cols, cols, None, cols, d, 0, 0.0, 1e-6, None, cols, d, cols, None, 0, None, 0,
                              0, None)
        assert rc == 1 and b"too many rows" in lib.gdn_last_error(), (rows, cols)


def test_layer_refuses_8_bit_rows_of_another_input():
    from logssms_amd.layers import GatedDeltaNet
    _built()
    net = GatedDeltaNet(64, 2, 4, 32, 32, 4, 1e-6, 0, device="cpu", dtype=torch.bfloat16)
    net.in_proj_qkvz_weight.zero_()
    net.out_proj_weight.zero_()
    net.quantize_weights()
    x = torch.zeros(5, 64, dtype=torch.bfloat16)
    for given in (_pair(4, 64), _pair(5, 48), _pair(1, 64)):
        with pytest.raises(AssertionError, match="x in 8 bits"):
            net.proj(x, given)
    with pytest.raises(AssertionError, match="tokens"):
        net.proj(x.view(5, 1, 64))


def test_product_refuses_what_its_offsets_cannot_reach():
    lib = _built()
    d = 0x10000

    def linear(M=4, N=64, xs=d, ws=d, ost=64):
        return lib.gdn_fp8_linear(d, 128, xs, 1, 4, d, 128, ws, 1, 1, M, N, 128, d, 1, ost, None)

    most = (1 << 31) - 4096
    for kw in (dict(M=most + 1), dict(N=most + 1, ost=most + 1), dict(M=1, N=1 << 40, ost=1 << 40),
               dict(ost=(1 << 22) + 1)):
        assert linear(**kw) == 2, kw
    for kw in (dict(xs=d + 2), dict(ws=d + 1)):
        assert linear(**kw) == 1 and b"misaligned scales" in lib.gdn_last_error(), kw


def test_weights_are_quantised_without_a_gradient():
    """A parameter's values and scales are data: they keep no graph of the weight alive."""
    from logssms_amd.kernel.fp8 import quantize_fp8_weight
    w = torch.nn.Parameter(torch.randn(130, 200, generator=_gen(4)))
    q = quantize_fp8_weight(w)
    assert not q.values.requires_grad and not q.scales.requires_grad and q.scales.grad_fn is None
    want = quantize_fp8_weight(w.detach())
    assert torch.equal(q.scales, want.scales) and torch.equal(q.dequantize(), want.dequantize())


def test_limits_of_strides_are_not_those_of_a_single_row():
    """Where there is more than one row, they are refused with the limits' own words."""
    lib = _built()
    d = 0x10000

    def linear(M, N, K, xst, wst, ost):
        return lib.gdn_fp8_linear(d, xst, d, 1, 4, d, wst, d, 1, 1, M, N, K, d, 1, ost, None)

    far = 1 << 24
    for kw in (dict(M=2, N=2, K=128, xst=128, wst=128, ost=(1 << 22) + 1),
               dict(M=2, N=2, K=128, xst=far, wst=128, ost=2), dict(M=2, N=2, K=128, xst=128, wst=far, ost=2),
               dict(M=1, N=2, K=far, xst=far, wst=far, ost=2)):
        assert linear(**kw) == 2, kw
        assert b"strides between rows" in lib.gdn_last_error()
