"""``GatedDeltaNet`` in 8 bits where the layer quantises its own input, and
where one of its weights is in 8 bits already."""

import pytest
import torch

from tests.gpu_util import DEV, gen, randn
from tests.test_gpu_layer import _layer

pytestmark = pytest.mark.gpu


def test_the_layer_quantises_its_own_input():
    """``forward(x)`` is ``forward(x, quantize_fp8(x))`` bit for bit, output and
    pools, in prefill and decode; other rows give other outputs."""
    from logssms_amd.cache import LinearStatePool
    from logssms_amd.core import Batch, Context, Request, clear_global_ctx, set_global_ctx
    from logssms_amd.kernel import quantize_fp8
    g = gen(292)
    hidden, H, HV, d = 192, 2, 4, 64
    net = _layer(g, hidden, H, HV, d, d, 0)
    net.quantize_weights()
    pool = LinearStatePool(24, 1, net.config.conv_dim, 4, HV, d, d, DEV, torch.bfloat16)
    pool.conv_state.copy_(randn(*pool.conv_state.shape, g=g, dtype=torch.bfloat16))
    pool.recurrent_state.copy_(randn(*pool.recurrent_state.shape, g=g, std=0.1))
    table = torch.tensor([[8 * i + p // 64 for p in range(384)] for i in range(3)], device=DEV)
    reqs = [(0, 0, 70), (1, 128, 200), (2, 64, 129)]  # (table row, cached, device_len)
    ctx = Context(page_size=64, linear_state=pool, state_table=table)
    set_global_ctx(ctx)
    try:
        for phase in ("prefill", "decode"):
            if phase == "prefill":
                batch = Batch(reqs=[Request(t, c, e) for t, c, e in reqs], phase="prefill")
            else:
                batch = Batch(reqs=[Request(t, e, e + 1) for t, _, e in reqs], phase="decode")
            n = sum(e - c for _, c, e in reqs) if phase == "prefill" else len(reqs)
            ctx.batch = batch
            ctx.linear_attn_backend.prepare_metadata(batch)
            x = randn(n, hidden, g=g, dtype=torch.bfloat16).to(DEV)
            start = pool.conv_state.clone(), pool.recurrent_state.clone()

            def run(*args):
                pool.conv_state.copy_(start[0])
                pool.recurrent_state.copy_(start[1])
                return net.forward(*args), pool.conv_state.clone(), pool.recurrent_state.clone()

            given = run(x, quantize_fp8(x))
            assert given[0].isfinite().all() and not torch.equal(given[2], start[1])
            other = run(x, quantize_fp8(x.flip(0)))
            assert not torch.equal(other[0], given[0]) and not torch.equal(other[1], given[1])
            own = run(x)  # last: its pools are the next phase's
            assert all(torch.equal(a, b) for a, b in zip(own, given))
    finally:
        clear_global_ctx()


def test_weights_that_are_in_8_bits_already_stay():
    net = _layer(gen(293), 64, 2, 4, 32, 32, 0)
    plain = net.in_proj_qkvz_weight
    net.quantize_weights()
    first, second = net.in_proj_qkvz_weight, net.out_proj_weight
    net.in_proj_qkvz_weight = plain
    net.quantize_weights()
    assert net.out_proj_weight is second and net.in_proj_qkvz_weight is not first
    assert torch.equal(net.in_proj_qkvz_weight.scales, first.scales)
    assert torch.equal(net.in_proj_qkvz_weight.dequantize(), first.dequantize())
