"""The block-scaled 8-bit product (``gdn_fp8_linear``, ``csrc/fp8_linear.hip``)
against ``oracle/fp8.py`` in float64 on the same quantised operands.  The bound
is the oracle's (``linear_bound``: what the 8-bit matrix instructions and fp32
sums may lose) plus half a step of the output's type."""

import pytest
import torch

from oracle import fp8 as ref
from tests.gpu_util import DEV, gen, randn

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}

#         M, N, K
SHAPES = [(1, 1, 1), (1, 16, 128), (2, 17, 130), (1, 2048, 4096), (16, 48, 256), (17, 100, 1000), (33, 128, 16),
          (64, 333, 272), (31, 200, 2048), (65, 129, 131), (129, 257, 384), (300, 1111, 1000), (256, 256, 128),
          (100, 64, 5000), (513, 130, 640), (200, 1, 33)]
ids = [f"{m}x{n}x{k}" for m, n, k in SHAPES]


def operands(m, n, k, g, wild=0.0):
    """Quantised operands whose blocks differ in size, with garbage (NaN codes)
    in the bytes behind each row's end."""
    wide = (k + 15) // 16 * 16

    def rows(count, scale_rows):
        v = randn(count, k, g=g, std=60.0) * torch.exp(wild * randn(count, k, g=g))
        codes = torch.full((count, wide), 0x7F, dtype=torch.uint8)
        codes[:, :k] = v.clamp(-448, 448).to(FP8).view(torch.uint8)
        scales = 0.01 * torch.exp(randn(scale_rows, -(-k // 128), g=g))
        return codes.view(FP8)[:, :k], scales

    return rows(m, m), rows(n, -(-n // 128))


def to_dev(pair):
    from logssms_amd.kernel import Fp8Tensor
    values, scales = pair
    count, k = values.shape
    wide = values.as_strided((count, values.stride(0)), (values.stride(0), 1))
    return Fp8Tensor(wide.to(DEV)[:, :k], scales.to(DEV))


def check(got, x, w, dtype, rows=None, cols=None):
    """got against the oracle on some rows and columns (all by default)."""
    rows = torch.arange(x[0].shape[0]) if rows is None else rows
    cols = torch.arange(w[0].shape[0]) if cols is None else cols
    k = x[0].shape[1]
    a = ref.dequantize(x[0], x[1])[rows].to(DEV)
    b = ref.dequantize(w[0], w[1])[cols].to(DEV)
    one = torch.ones(1, -(-k // 128), dtype=torch.float64, device=DEV)
    want = a @ b.t()
    loss = ref.linear_bound(a, one.expand(len(rows), -1), b, one.expand(len(cols), -1))
    assert got.dtype == dtype
    err = (got[rows.to(DEV)][:, cols.to(DEV)].double() - want).abs()
    bound = loss + (want.abs() + loss) * HALF[dtype] + FLOOR[dtype]
    assert (err <= bound).all(), f"{float((err / bound).max())} times the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_product_matches_oracle(shape, dtype):
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    m, n, k = shape
    print(f"fp8_linear {shape} {dtype}", flush=True)
    for wild in (0.0, 1.5):
        x, w = operands(m, n, k, gen(m + n + k), wild)
        dx, dw = to_dev(x), to_dev(w)
        got = fp8_linear(dx, dw, dtype)
        assert got.shape == (m, n)
        check(got, x, w, dtype)
        # the scales of the tokens block by block, as the quantisers lay them out
        again = fp8_linear(Fp8Tensor(dx.values, dx.scales.t().contiguous().t()), dw, dtype)
        assert torch.equal(again, got)


@pytest.mark.parametrize("shape", [(4096, 4097, 160), (5000, 4000, 1040), (700, 6000, 2050), (16, 12288, 2048)],
                         ids=str)
def test_large_products_on_sampled_rows(shape):
    from logssms_amd.kernel import fp8_linear
    m, n, k = shape
    print(f"fp8_linear large {shape}", flush=True)
    g = gen(m)
    x, w = operands(m, n, k, g, 0.5)
    got = fp8_linear(to_dev(x), to_dev(w))
    rows = torch.unique(torch.cat([torch.arange(min(m, 40)), torch.randint(0, m, (160,), generator=g),
                                   torch.arange(max(0, m - 40), m)]))
    cols = torch.unique(torch.cat([torch.arange(40), torch.randint(0, n, (160,), generator=g), torch.arange(n - 40, n)]))
    check(got, x, w, torch.bfloat16, rows, cols)
    # every element, against the fp32 product of the dequantised operands
    want = (ref.dequantize(*x).to(DEV) @ ref.dequantize(*w).to(DEV).t()).float()
    rms = want.square().mean().sqrt()
    assert ((got.float() - want).abs() <= 2.0 ** -7 * (want.abs() + rms)).all()


@pytest.mark.parametrize("m", [1, 40, 300])
def test_strides_and_untouched_surroundings(m):
    """Operands and output inside larger buffers; what lies around the output stays."""
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    n, k = 200, 272
    print(f"fp8_linear strides m={m}", flush=True)
    g = gen(m)
    x, w = operands(m, n, k, g)
    dx, dw = to_dev(x), to_dev(w)
    plain = fp8_linear(dx, dw)
    wide = torch.full((m + 2, 512), 0x7F, dtype=torch.uint8, device=DEV).view(FP8)
    wide.view(torch.uint8)[1:m + 1, 64:64 + k] = dx.values.view(torch.uint8)
    scales = torch.full((m + 2, 8), float("nan"), device=DEV)
    scales[1:m + 1, 1:7:2] = dx.scales
    weight = torch.full((n + 2, 304), 0x7F, dtype=torch.uint8, device=DEV).view(FP8)
    weight.view(torch.uint8)[2:, 16:16 + k] = dw.values.view(torch.uint8)
    for pad in (3, 8):  # rows of the output at odd addresses and at multiples of 16 bytes
        out = torch.full((m + 2, n + 2 * pad), 7.0, dtype=torch.bfloat16, device=DEV)
        view = out[1:m + 1, pad:pad + n]
        got = fp8_linear(Fp8Tensor(wide[1:m + 1, 64:64 + k], scales[1:m + 1, 1:7:2]),
                         Fp8Tensor(weight[2:, 16:16 + k], dw.scales.t().contiguous().t()), out=view)
        assert got is view and torch.equal(view, plain)
        view.fill_(7.0)
        assert (out == 7.0).all()


@pytest.mark.parametrize("m", [3, 50, 200])
def test_what_is_not_finite_stays_in_its_row_or_column(m):
    from logssms_amd.kernel import fp8_linear
    n, k = 150, 300
    print(f"fp8_linear nan m={m}", flush=True)
    x, w = operands(m, n, k, gen(m))
    x[0].view(torch.uint8)[1, 299] = 0x7F
    x[1][2, 0] = float("inf")
    w[0].view(torch.uint8)[149, 0] = 0xFF
    got = fp8_linear(to_dev(x), to_dev(w)).cpu()
    assert got[1].isnan().all() and not got[2, :149].isfinite().any() and got[:, 149].isnan().all()
    rest = torch.ones(m, n, dtype=torch.bool)
    rest[1], rest[2], rest[:, 149] = False, False, False
    assert got[rest].isfinite().all()


@pytest.mark.parametrize("m", [5, 90, 600])
def test_same_bits_every_time_and_for_every_batch(m):
    """A row's result does not depend on the call, on other work, or (within a
    form of the kernel) on the rows beside it."""
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    x, w = operands(m, 700, 1000, gen(m))
    dx, dw = to_dev(x), to_dev(w)
    first = fp8_linear(dx, dw)
    for _ in range(3):
        assert torch.equal(fp8_linear(dx, dw), first)
    perm = torch.randperm(m, generator=gen(1)).to(DEV)
    shuffled = Fp8Tensor(to_dev((x[0].as_strided((m, 1008), (1008, 1)), x[1])).values.view(torch.uint8)[perm].view(FP8)[:, :1000],
                         dx.scales[perm])
    assert torch.equal(fp8_linear(shuffled, dw), first[perm])


@pytest.mark.parametrize("m", [1, 48, 300])
def test_norms_and_products_in_one_graph(m):
    """The run of a layer: residual norm in 8 bits, product, gated norm in 8
    bits, product; captured and replayed on new inputs beside eager work."""
    from logssms_amd.kernel import add_rms_norm_fp8, fp8_linear, quantize_fp8_weight, rms_norm_gated_fp8
    g = gen(m)
    hidden, heads = 256, 4
    x, res = (randn(m, hidden, g=g, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    weight = (1 + 0.1 * randn(hidden, g=g)).to(DEV)
    head_weight = (1 + 0.1 * randn(128, g=g)).to(DEV)
    w_in = quantize_fp8_weight(randn(2 * heads * 128, hidden, g=g, std=0.06).to(DEV))
    w_out = quantize_fp8_weight(randn(hidden, heads * 128, g=g, std=0.04).to(DEV))

    def layer():
        q, total = add_rms_norm_fp8(x, res, weight, 1e-6)
        core, z = fp8_linear(q, w_in).view(m, 2 * heads, 128).split(heads, 1)
        p = rms_norm_gated_fp8(core, z, head_weight, 1e-6)
        return q, core, z, p, fp8_linear(p, w_out), total

    def expected(q, core, z, p):
        _, y = ref.rms_norm(x.cpu(), weight.cpu(), 1e-6, residual=res.cpu())
        first = ref.linear(q.values.cpu(), q.scales.cpu(), w_in.values.cpu(), w_in.scales.cpu())
        gated = ref.rms_norm_gated(core.cpu(), z.cpu(), head_weight.cpu(), 1e-6)
        last = ref.linear(p.values.cpu(), p.scales.cpu(), w_out.values.cpu(), w_out.scales.cpu())
        return y, first, gated, last

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed = layer()
    for _ in range(3):
        x.copy_(randn(m, hidden, g=g, dtype=torch.bfloat16).to(DEV))
        q, core, z, p, out, total = layer()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphed[4], out) and torch.equal(graphed[5], total)
        y, first, gated, last = expected(q, core, z, p)
        # each step against the oracle on the step's own inputs: a code's half step,
        # and 2^-7 of the row's size for a product rounded to bf16
        assert ((q.dequantize().double().cpu() - y).abs() <= 2.0 ** -4 * 1.01 * y.abs() + 2.0 ** -10 * 0.02).all()
        both = torch.cat([core, z], 1).flatten(1).double().cpu()
        for got, want in ((both, first), (out.double().cpu(), last)):
            assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * want.square().mean().sqrt() * 8).all()
        assert ((p.dequantize().double().cpu() - gated).abs()
                <= 2.0 ** -4 * 1.01 * gated.abs() + 2.0 ** -10 * 0.02).all()


# tokens, columns: a size for each form and tile of the kernel, none of them a multiple of the tile
FORMS = [(5, 270), (9, 5003), (16, 33001), (45, 2050), (100, 1500), (30, 9001), (120, 4001), (64, 20001), (130, 6001),
         (450, 8003), (700, 6002), (1530, 2050), (4090, 4093)]


@pytest.mark.parametrize("k", [7, 128, 255, 384, 1041])
@pytest.mark.parametrize("size", FORMS, ids=str)
def test_every_form_with_its_tails(size, k):
    """Each form of the kernel with one block of K and several, whole and not;
    the output lies in a larger buffer whose other values stay."""
    from logssms_amd.kernel import fp8_linear
    m, n = size
    print(f"fp8_linear form {size} {k}", flush=True)
    g = gen(m + k)
    x, w = operands(m, n, k, g, 0.5)
    dx, dw = to_dev(x), to_dev(w)
    rows = torch.unique(torch.cat([torch.arange(min(m, 40)), torch.randint(0, m, (100,), generator=g),
                                   torch.arange(max(0, m - 40), m)]))
    cols = torch.unique(torch.cat([torch.arange(min(n, 40)), torch.randint(0, n, (100,), generator=g),
                                   torch.arange(max(0, n - 40), n)]))
    got = fp8_linear(dx, dw)
    check(got, x, w, torch.bfloat16, rows, cols)
    a, b = ref.dequantize(*x).to(DEV), ref.dequantize(*w).to(DEV)
    # every element: by the oracle's bound at most 7 * 2^-12 of the sum of the
    # products' sizes is lost, and 2^-15 of it in the fp32 sums of these K; both,
    # with the rounding of them, are below 2^-9; half a step of the output
    size_of, want = a.abs() @ b.abs().t(), a @ b.t()
    for pad in (3, 8):
        out = torch.full((m + 2, (n + 2 * pad + 7) // 8 * 8), 7.0, dtype=torch.bfloat16, device=DEV)
        view = out[1:m + 1, pad:pad + n]
        assert fp8_linear(dx, dw, out=view) is view
        assert torch.equal(view, got)
        assert ((view.double() - want).abs() <= 2.0 ** -9 * size_of + 2.0 ** -8 * want.abs() + 2.0 ** -134).all()
        view.fill_(7.0)
        assert (out == 7.0).all()


@pytest.mark.parametrize("size", FORMS, ids=str)
def test_every_form_keeps_rows_and_columns_apart(size):
    """NaN codes and infinite scales reach their own row or column only, and a
    row's bits do not depend on its place among the others."""
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    m, n = size
    k = 300
    print(f"fp8_linear apart {size}", flush=True)
    x, w = operands(m, n, k, gen(m))
    dx, dw = to_dev(x), to_dev(w)
    clean = fp8_linear(dx, dw)
    perm = torch.randperm(m, generator=gen(1)).to(DEV)
    codes = dx.values.view(torch.uint8).as_strided((m, 304), (304, 1))[perm].view(FP8)[:, :k]
    assert torch.equal(fp8_linear(Fp8Tensor(codes, dx.scales[perm]), dw), clean[perm])
    row, col = m // 2, n - 1 - n // 3
    dx.values.view(torch.uint8)[row, k - 1] = 0x7F
    dx.scales[m - 1, 1] = float("inf")
    dw.values.view(torch.uint8)[col, 0] = 0xFF
    got = fp8_linear(dx, dw)
    assert got[row].isnan().all() and got[:, col].isnan().all() and not got[m - 1].isfinite().any()
    got[row], got[m - 1], got[:, col] = clean[row], clean[m - 1], clean[:, col]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("size", [(66000, 40000, 48), (3, 270000, 16400), (270000, 3, 16400), (70000, 500, 65000)],
                         ids=str)
def test_offsets_beyond_32_bits(size):
    """Weights, tokens and outputs of more than 2^32 bytes, checked at their ends."""
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    m, n, k = size
    print(f"fp8_linear far {size}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(m + n)
    kb = -(-k // 128)

    def made(count, scale_rows):
        wide = (k + 15) // 16 * 16
        codes = torch.randint(0, 256, (count, wide), generator=g, device=DEV, dtype=torch.uint8)
        codes &= 0xBF  # below 2: no NaN codes, and sums far from overflow
        return Fp8Tensor(codes.view(FP8)[:, :k], 0.5 + torch.rand(kb, scale_rows, generator=g, device=DEV).t())

    x, w = made(m, m), made(n, -(-n // 128))
    got = fp8_linear(x, w)
    rows = torch.unique(torch.cat([torch.arange(min(m, 20)), torch.arange(max(0, m - 40), m)])).to(DEV)
    cols = torch.unique(torch.cat([torch.arange(min(n, 20)), torch.arange(max(0, n - 40), n)])).to(DEV)
    # the sampled rows of the weights carry their blocks' scales as rows of their own
    a = (x.values.view(torch.uint8)[rows].view(FP8).cpu(), x.scales[rows].cpu())
    b = w.values.view(torch.uint8)[cols].view(FP8).cpu(), w.scales[cols // 128].cpu()
    va, vb = ref.dequantize(*a), ref.dequantize(*b)
    want, size_of = va @ vb.t(), va.abs() @ vb.abs().t()
    # the oracle's bound: 7 * 2^-12 of the products' sizes, and K / 8 + K / 128 + 2
    # additions of 2^-23 of them; half a step of bf16
    err = (got[rows][:, cols].cpu().double() - want).abs()
    assert (err <= (2.0 ** -8 * want.abs() + (2.0 ** -9 + (k / 8 + k / 128 + 2) * 2.0 ** -23) * 1.01 * size_of)).all()


@pytest.mark.parametrize("k", [30, 128, 1041, 2600])
@pytest.mark.parametrize("size", [(140, 5003), (190, 5001), (131, 5900), (200, 8001), (16000, 40), (9000, 20),
                                  (5000, 130)], ids=str)
def test_forms_between_and_narrow_outputs(size, k):
    """48 x 64, 64 x 64 and 64 x 80 outputs a block, 64 x 128 of more than 64
    rows, and outputs that are narrower than a tile."""
    test_every_form_with_its_tails(size, k)
    if k == 1041:
        test_every_form_keeps_rows_and_columns_apart(size)
