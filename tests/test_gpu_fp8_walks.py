"""The block-scaled product where a block of the kernel walks over several
output tiles, and what one tile may leave for the next: scales that are not
finite, tails of K, narrow stores.  Bounds as in ``test_gpu_fp8_linear``."""

import pytest
import torch

from tests.gpu_util import DEV, gen
from tests.test_gpu_fp8_linear import operands, test_every_form_keeps_rows_and_columns_apart as keeps_apart
from tests.test_gpu_fp8_linear import test_every_form_with_its_tails as form_with_its_tails
from tests.test_gpu_fp8_linear import to_dev

pytestmark = pytest.mark.gpu

# tokens, columns: more tiles than blocks for 64 x 128 outputs a block (four
# stages; two and three tiles a block), 128 x 128 two to a CU and 256 x 256
WALKS = [(40, 40001), (64, 70000), (4097, 4099), (4090, 8003)]
# one tile a block, or a form without tiles
SINGLE = [(9, 5003), (60, 2050), (64, 20001), (130, 6001), (700, 6002)]


@pytest.mark.parametrize("value", [float("inf"), float("nan")], ids=str)
@pytest.mark.parametrize("size", WALKS + SINGLE, ids=str)
def test_a_weight_scale_that_is_not_finite_stays_in_its_block(size, value):
    """In the last block of K of an early column block: its 128 columns change, nothing else."""
    from logssms_amd.kernel import fp8_linear
    m, n = size
    print(f"fp8_linear weight scale {size} {value}", flush=True)
    x, w = operands(m, n, 300, gen(m + n))
    dx, dw = to_dev(x), to_dev(w)
    clean = fp8_linear(dx, dw)
    assert clean.isfinite().all()
    for block in (0, 5):
        keep = dw.scales[block, -1].clone()
        dw.scales[block, -1] = value
        got = fp8_linear(dx, dw)
        dw.scales[block, -1] = keep
        part = slice(128 * block, 128 * block + 128)
        assert not got[:, part].isfinite().any()
        got[:, part] = clean[:, part]
        assert torch.equal(got, clean)


def test_a_single_row_has_no_stride_to_limit():
    """One token by more than 2^22 columns, and one token by one column over more
    than 2^23 of K: the stride of a single row means nothing.  Sums of small whole
    numbers, exact in any order; above 256 they are rounded to bf16 once."""
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    fp8 = torch.float8_e4m3fn
    g = torch.Generator(device=DEV).manual_seed(1)

    def whole(rows, k):
        v = torch.randint(-2, 3, (rows, -(-k // 16) * 16), generator=g, device=DEV, dtype=torch.int8)
        return v.bfloat16().to(fp8)[:, :k]

    for n, k in (((1 << 22) + 1, 128), ((1 << 22) + 24, 40), (1, (1 << 23) + 16), (1, (1 << 23) + 1001)):
        print(f"fp8_linear single row 1 x {n} x {k}", flush=True)
        x, w = whole(1, k), whole(n, k)
        blocks = -(-k // 128)
        got = fp8_linear(Fp8Tensor(x, torch.ones(1, blocks, device=DEV)),
                         Fp8Tensor(w, torch.ones(-(-n // 128), blocks, device=DEV)))
        # the hardware drops nothing: products of a group are at most 4 and at least 1 apart from zero
        want = (w.float() * x.float()).sum(1) if k < 1000 else (w.double() * x.double()).sum(1).float()
        assert torch.equal(got, want.bfloat16()[None])


@pytest.mark.parametrize("k", [7, 128, 255, 1041])
@pytest.mark.parametrize("size", WALKS, ids=str)
def test_several_tiles_a_block_with_their_tails(size, k):
    """The turn to the next tile, the end of K in its first step, the scaling that
    a step leaves to the next, wide and narrow stores behind one another."""
    form_with_its_tails(size, k)


@pytest.mark.parametrize("size", WALKS, ids=str)
def test_several_tiles_a_block_keep_rows_and_columns_apart(size):
    keeps_apart(size)


@pytest.mark.parametrize("k", [7, 300, 1041])
@pytest.mark.parametrize("m", [1, 300, 9000, 20000, 70000])
def test_a_single_column(m, k):
    """One row of weights, in the forms for few tokens and in each tile that so many tokens take."""
    form_with_its_tails((m, 1), k)


def test_strides_of_single_rows_are_not_read():
    """Operands, scales and output of one row at strides that no row could have."""
    from logssms_amd.kernel import Fp8Tensor, fp8_linear
    for m, n in ((1, 200), (40, 1), (1, 1)):
        print(f"fp8_linear strides of single rows {m} x {n}", flush=True)
        x, w = operands(m, n, 272, gen(m + n))
        dx, dw = to_dev(x), to_dev(w)
        want = fp8_linear(dx, dw)

        def odd(t, stride):
            return t.as_strided(t.shape, (stride, t.stride(1))) if t.shape[0] == 1 else t

        for stride in (0, 3, 1 << 40):
            out = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
            got = fp8_linear(Fp8Tensor(odd(dx.values, stride), odd(dx.scales, stride)),
                             Fp8Tensor(odd(dw.values, stride), odd(dw.scales, stride)), out=odd(out, stride))
            assert torch.equal(got, want) and torch.equal(out, want)
