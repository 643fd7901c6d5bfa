"""Norms with the residual's addition and 8-bit outputs, and the quantisation of
rows (``gdn_rms_norm``, ``gdn_quantize_fp8``, ``gdn_rms_norm_gated_fp8``,
``csrc/rms_norm.hip``), against ``oracle/fp8.py`` in float64.

Tolerances, from the operations: a sum of squares runs over at most 512 terms
per lane and ten joining additions, each off by 2^-24 of a positive sum; half
of that relative error reaches the norm, then rsqrt, exp and a handful of
products at 2^-23 each: under (522 / 2 + 16) * 2^-24 < 2^-15 of the value.  A
stored result adds half a step of its type, a code half a step of e4m3."""

import pytest
import torch

from oracle import fp8 as ref
from tests.gpu_util import DEV, gen, randn

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
DELTA = 2.0 ** -15
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the least step
EPS = 1e-6

SHAPES = [(1, 1), (3, 7), (5, 16), (9, 130), (130, 64), (4, 128), (1, 2048), (37, 1000), (6, 1024), (3, 2056),
          (2, 4096), (2, 8192), (3, 8200), (2, 20001), (700, 2048)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ids = [f"{r}x{c}" for r, c in SHAPES]


def assert_rounded(got, want, dtype):
    """A value computed in fp32 and rounded once to dtype."""
    assert got.dtype == dtype
    err = (got.double().cpu() - want).abs()
    assert (err <= want.abs() * (HALF[dtype] + 2 * DELTA) + FLOOR[dtype]).all(), float((err / want.abs()).max())


def assert_quantised(q, want):
    """Scales near max|block| / 448, codes half a step from value / scale."""
    rows, cols = want.shape
    values, scales = q.values.cpu(), q.scales.cpu()
    assert values.dtype == FP8 and values.shape == (rows, cols)
    assert scales.dtype == torch.float32 and scales.shape == (rows, -(-cols // 128))
    s64 = ref.block_scales(want)
    assert ((scales.double() - s64).abs() <= 2 * DELTA * s64).all()
    err = (ref.dequantize(values, scales) - want).abs()
    bound = want.abs() * (ref.HALF_STEP + 3 * DELTA) + ref.spread(s64, rows, cols) * 1.001 * ref.HALF_STEP_SUBNORMAL
    assert (err <= bound).all(), float((err - bound).max())
    if cols % 16 and rows:  # the row's last 16 bytes are zeros past its end
        wide = q.values.as_strided((rows, (cols + 15) // 16 * 16), q.values.stride())
        assert (wide.view(torch.uint8)[:, cols:] == 0).all()


def _rows(rows, cols, dtype, g, strided):
    if not strided:
        return randn(rows, cols, g=g, dtype=dtype).to(DEV)
    return randn(rows, cols + 24, g=g, dtype=dtype).to(DEV)[:, 8:8 + cols]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_norm_without_and_with_residual(shape, dtype):
    from logssms_amd.kernel import add_rms_norm, add_rms_norm_fp8, rms_norm, rms_norm_fp8
    rows, cols = shape
    print(f"rms_norm {shape} {dtype}", flush=True)
    g = gen(1000 * rows + cols)
    for strided, wdt, offset in ((False, torch.float32, 0.0), (True, dtype, 1.0)):
        x, res = (_rows(rows, cols, dtype, g, strided) for _ in range(2))
        w = randn(cols, g=g, std=0.5).to(wdt).to(DEV)
        h, y = ref.rms_norm(x.cpu(), w.cpu(), EPS, weight_offset=offset)
        assert_rounded(rms_norm(x, w, EPS, weight_offset=offset), y, dtype)
        q, kept = rms_norm_fp8(x, w, EPS, weight_offset=offset, keep=True)
        assert_quantised(q, y)
        assert_rounded(kept, y, dtype)
        h, y = ref.rms_norm(x.cpu(), w.cpu(), EPS, residual=res.cpu(), weight_offset=offset)
        total = (x.float() + res.float()).to(dtype)  # one rounding of the fp32 sum
        got, got_sum = add_rms_norm(x, res, w, EPS, weight_offset=offset)
        assert_rounded(got, y, dtype)
        assert torch.equal(got_sum, total)
        q, got_sum = add_rms_norm_fp8(x, res, w, EPS, weight_offset=offset)
        assert_quantised(q, y)
        assert torch.equal(got_sum, total)
        both, in_place = add_rms_norm(x, res, w, EPS, weight_offset=offset, residual_out=res)
        assert in_place is res and torch.equal(res, total) and torch.equal(both, got)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_quantised_rows(shape, dtype):
    from logssms_amd.kernel import quantize_fp8
    rows, cols = shape
    print(f"quantize {shape} {dtype}", flush=True)
    g = gen(rows + 7 * cols)
    for strided in (False, True):
        x = _rows(rows, cols, dtype, g, strided)
        assert_quantised(quantize_fp8(x), x.double().cpu())
    x = randn(2, rows, cols, g=g, dtype=dtype).to(DEV)
    assert_quantised(quantize_fp8(x), x.double().cpu().view(-1, cols))
    t = randn(cols, rows, g=g, dtype=dtype).to(DEV).t()  # no unit column stride: copied
    assert_quantised(quantize_fp8(t), t.double().cpu())


def test_equal_to_torch_on_exact_scales():
    """With the largest value of each block at 448 the scale is 1 and the codes are torch's."""
    from logssms_amd.kernel import quantize_fp8
    g = gen(5)
    x = (randn(64, 512, g=g) * torch.exp(3 * randn(64, 512, g=g))).clamp(-448, 448)
    x[:, ::128] = 448.0
    q = quantize_fp8(x.to(DEV))
    assert (q.scales == 1).all()
    assert torch.equal(q.values.cpu().view(torch.uint8), x.to(FP8).view(torch.uint8))


def test_blocks_of_zeros_tiny_values_and_what_is_not_finite():
    from logssms_amd.kernel import quantize_fp8, rms_norm_fp8
    x = torch.zeros(5, 384)
    x[1, 0], x[1, 200], x[2, 130] = float("nan"), 3.0, float("inf")
    x[3, 5], x[3, 300] = 2.0 ** -130, -1e-30
    x[4, :] = 3.0e38
    q = quantize_fp8(x.to(DEV))
    d = ref.dequantize(q.values.cpu(), q.scales.cpu())
    assert (d[0] == 0).all() and (q.scales[0] == 2.0 ** -126).all()
    # 448 times the fp32 scale is the block's largest value up to the scale's rounding, 2^-24 of it
    assert d[1, :128].isnan().all() and abs(float(d[1, 200]) - 3.0) <= 3.0 * 2.0 ** -24 and (d[1, 256:] == 0).all()
    assert (d[2, :128] == 0).all() and d[2, 128:256].isnan().all() and (d[2, 256:] == 0).all()
    assert abs(float(d[3, 5]) - 2.0 ** -130) <= 2.0 ** -134 and float(d[3, 300]) == pytest.approx(-1e-30, rel=1e-6)
    assert ((d[4] - x[4].double()).abs() <= 2.0 ** -23 * x[4].double()).all()
    # a row of zeros normalises to zeros; a NaN spreads over its own row alone
    x = torch.zeros(3, 384, dtype=torch.bfloat16)
    x[1, 7], x[2] = float("nan"), 1.0
    w = torch.ones(384)
    q, y = rms_norm_fp8(x.to(DEV), w.to(DEV), EPS, keep=True)
    d = ref.dequantize(q.values.cpu(), q.scales.cpu())
    assert (d[0] == 0).all() and (y[0] == 0).all()
    assert d[1].isnan().all() and y[1].isnan().all()
    assert ((d[2] - 1).abs() <= 2.0 ** -4).all() and (y[2] == 1).all()


def test_weights_that_are_not_finite_stay_in_their_columns():
    """A column past the row's end is a zero of the block, whatever the offset."""
    from logssms_amd.kernel import rms_norm_fp8
    x = randn(4, 130, g=gen(8), dtype=torch.bfloat16)
    w = torch.ones(130)
    w[129] = float("inf")
    q, y = rms_norm_fp8(x.to(DEV), w.to(DEV), EPS, weight_offset=float("1.0"), keep=True)
    d = ref.dequantize(q.values.cpu(), q.scales.cpu())
    assert d[:, :128].isfinite().all() and d[:, 128:].isnan().all()
    assert y[:, :129].isfinite().all() and y[:, 129].isinf().all()


GATED = [(1, 32, 128), (7, 3, 96), (5, 4, 32), (3, 2, 256), (2, 1, 512), (4, 5, 64), (3, 3, 8), (2, 2, 100), (3, 7, 16),
         (1, 1, 1), (2, 300, 24), (600, 32, 128)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", GATED, ids=[f"t{t}_h{h}_d{d}" for t, h, d in GATED])
def test_gated_norm_in_8_bits(case, dtype):
    from logssms_amd.kernel import rms_norm_gated_fp8
    tokens, heads, dim = case
    print(f"gated {case} {dtype}", flush=True)
    g = gen(tokens + 10 * heads + 100 * dim)
    x = randn(tokens, heads, dim, g=g, dtype=dtype)
    z = randn(tokens, heads * dim + 40, g=g, dtype=dtype)[:, 8:8 + heads * dim].view(tokens, heads, dim)
    for wdt in (torch.float32, torch.bfloat16):
        w = randn(dim, g=g, std=0.5).to(wdt)
        got = rms_norm_gated_fp8(x.to(DEV), z.to(DEV), w.to(DEV), EPS)
        assert_quantised(got, ref.rms_norm_gated(x, z, w, EPS))
    # heads and channels in another order in memory
    xt = randn(heads, tokens, dim, g=g, dtype=dtype).transpose(0, 1)
    zt = randn(dim, tokens, heads, g=g, dtype=dtype).permute(1, 2, 0)
    got = rms_norm_gated_fp8(xt.to(DEV), zt.to(DEV), w.to(DEV), EPS)
    assert_quantised(got, ref.rms_norm_gated(xt, zt, w, EPS))


def test_no_rows():
    from logssms_amd.kernel import add_rms_norm_fp8, quantize_fp8, rms_norm, rms_norm_gated_fp8
    x = torch.empty(0, 200, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(200, device=DEV)
    assert rms_norm(x, w, EPS).shape == (0, 200)
    q, total = add_rms_norm_fp8(x, x, w, EPS)
    assert q.values.shape == (0, 200) and q.scales.shape == (0, 2) and total.shape == (0, 200)
    assert quantize_fp8(x).values.shape == (0, 200)
    assert rms_norm_gated_fp8(x.view(0, 2, 100), x.view(0, 2, 100), w[:100], EPS).values.shape == (0, 200)


def test_rows_around_the_destination_stay():
    """A residual inside a larger buffer: only its rows and columns change."""
    from logssms_amd.kernel import add_rms_norm
    g = gen(21)
    big = randn(9, 300, g=g, dtype=torch.bfloat16).to(DEV)
    before = big.clone()
    x = randn(5, 200, g=g, dtype=torch.bfloat16).to(DEV)
    part = big[2:7, 40:240]
    add_rms_norm(x, part, torch.ones(200, device=DEV), EPS, residual_out=part)
    assert torch.equal(part, (x.float() + before[2:7, 40:240].float()).bfloat16())
    big[2:7, 40:240] = before[2:7, 40:240]
    assert torch.equal(big, before)


def test_rows_graph_replay_on_a_side_stream():
    from logssms_amd.kernel import add_rms_norm_fp8, quantize_fp8, rms_norm_gated_fp8
    g = gen(31)
    x = randn(33, 512, g=g, dtype=torch.bfloat16).to(DEV)
    res = randn(33, 512, g=g, dtype=torch.bfloat16).to(DEV)
    w = randn(512, g=g).to(DEV)

    def work():
        q, y, total = add_rms_norm_fp8(x, res, w, EPS, keep=True)
        p = rms_norm_gated_fp8(y.view(33, 4, 128), total.view(33, 4, 128), w[:128], EPS)
        return [*q, y, total, *p, *quantize_fp8(total)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eager = work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed = work()
    for i in range(4):
        if i:
            x.copy_(randn(33, 512, g=g, dtype=torch.bfloat16).to(DEV))
            eager = work()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(graphed, eager):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_rows_beyond_32_bits():
    """Rows whose offsets pass 2^32 bytes: the last ones are what they are alone."""
    from logssms_amd.kernel import add_rms_norm_fp8, quantize_fp8, rms_norm_gated_fp8
    rows, cols = 300000, 8192
    print("far rows", flush=True)
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    res = torch.empty_like(x).normal_(generator=g)
    weight = 1 + 0.1 * torch.randn(cols, generator=g, device=DEV)
    last = slice(rows - 5, rows)
    q, y, total = add_rms_norm_fp8(x, res, weight, 1e-6, keep=True)
    q1, y1, total1 = add_rms_norm_fp8(x[last], res[last], weight, 1e-6, keep=True)
    assert torch.equal(y[last], y1) and torch.equal(total[last], total1) and torch.equal(q.scales[last], q1.scales)
    assert torch.equal(q.values[last].view(torch.uint8), q1.values.view(torch.uint8))
    heads, heads_res, w128 = x.view(rows, 64, 128), res.view(rows, 64, 128), weight[:128].contiguous()
    for far, alone in ((quantize_fp8(x), quantize_fp8(x[last])),
                       (rms_norm_gated_fp8(heads, heads_res, w128, 1e-6),
                        rms_norm_gated_fp8(heads[last], heads_res[last], w128, 1e-6))):
        assert torch.equal(far.scales[last], alone.scales)
        assert torch.equal(far.values[last].view(torch.uint8), alone.values.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(5, 2157), (4, 2600), (3, 4801), (3, 6136), (2, 9001), (7, 333), (40, 12)], ids=str)
def test_rows_at_odd_addresses(shape, dtype):
    """Rows, residual and its destination at odd addresses and strides, in place;
    what lies beside the destination stays."""
    from logssms_amd.kernel import add_rms_norm, add_rms_norm_fp8, quantize_fp8
    rows, cols = shape
    print(f"odd rows {shape} {dtype}", flush=True)
    g = gen(rows + 7 * cols)
    wide = randn(3, rows + 1, cols + 5, g=g, dtype=dtype).to(DEV)
    x, res = wide[0][1:, 3:3 + cols], wide[1][1:, 1:1 + cols]
    w = randn(cols + 1, g=g).to(DEV)[1:]
    h, y = ref.rms_norm(x.cpu(), w.cpu(), EPS, residual=res.cpu(), weight_offset=1.0)
    around = wide[1].clone()
    got, total = add_rms_norm(x, res, w, EPS, weight_offset=1.0)
    assert_rounded(got, y, dtype)
    assert_rounded(total, h, dtype)
    assert_quantised(quantize_fp8(x), x.double().cpu())
    q, y8, place = add_rms_norm_fp8(x, res, w, EPS, weight_offset=1.0, keep=True, residual_out=res)
    assert_quantised(q, y)
    assert torch.equal(y8, got) and place is res and torch.equal(res, total)
    wide[1][1:, 1:1 + cols] = around[1:, 1:1 + cols]
    assert torch.equal(wide[1], around)


@pytest.mark.parametrize("case", [(3, 5, 96), (2, 3, 200), (3, 40, 96), (2, 10, 200), (2, 9, 130), (5, 4, 7),
                                  (1, 16384, 2)], ids=str)
def test_gated_heads_of_any_width(case):
    """One wave and four to a token, 16 and 64 lanes to a head, heads at odd addresses."""
    test_gated_norm_in_8_bits(case, torch.bfloat16)
    from logssms_amd.kernel import rms_norm_gated_fp8
    tokens, heads, dim = case
    g = gen(tokens + heads + dim)
    wide = randn(2, tokens, heads, dim + 3, g=g, dtype=torch.float16)
    x, z = wide[0][..., 1:1 + dim], wide[1][..., 2:2 + dim]
    w = randn(dim, g=g, std=0.5).half()
    on = wide.to(DEV)
    got = rms_norm_gated_fp8(on[0][..., 1:1 + dim], on[1][..., 2:2 + dim], w.to(DEV), EPS)
    assert_quantised(got, ref.rms_norm_gated(x, z, w, EPS))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("cols", [7, 200, 2056, 9001, 17000, 20001])
def test_the_sum_may_take_the_place_of_x(cols, dtype):
    """``residual_out`` is ``x``: every form of the norm, aligned and not, rows inside a larger buffer."""
    from logssms_amd.kernel import add_rms_norm, add_rms_norm_fp8
    g = gen(cols)
    w = randn(cols, g=g).to(DEV)
    for start in (0, 3):
        wide = randn(6, cols + 8, g=g, dtype=dtype).to(DEV)
        x, res = wide[1:, start:start + cols], randn(5, cols, g=g, dtype=dtype).to(DEV)
        kept, before = x.clone(), wide.clone()
        q1, y1, total = add_rms_norm_fp8(kept, res, w, EPS, keep=True)
        assert torch.equal(total, (kept.float() + res.float()).to(dtype))
        y, place = add_rms_norm(x, res, w, EPS, residual_out=x)
        assert place is x and torch.equal(x, total) and torch.equal(y, y1)
        x.copy_(kept)
        q, y, place = add_rms_norm_fp8(x, res, w, EPS, keep=True, residual_out=x)
        assert place is x and torch.equal(x, total) and torch.equal(y, y1)
        assert torch.equal(q.scales, q1.scales) and torch.equal(q.dequantize(), q1.dequantize())
        x.copy_(kept)
        assert torch.equal(wide, before)
