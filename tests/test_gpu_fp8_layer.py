"""``GatedDeltaNet`` with its large projections in block-scaled 8 bits: prefill
and decode through the backend, each stage against the oracle on the stage's
own inputs, the residual norm in front, and a captured decode step."""

import pytest
import torch

from oracle import fp8 as f8
from oracle import gdn as ref
from oracle import metadata as md
from tests.gpu_util import DEV, assert_state_close, gen, randn
from tests.test_gpu_fp8_linear import check
from tests.test_gpu_fp8_rows import DELTA, assert_quantised
from tests.test_gpu_layer import _layer

pytestmark = pytest.mark.gpu


def _host(q):
    return q.values.cpu(), q.scales.cpu()


def _check_output(net, core, z, y):
    """y against the unquantised gated norm times the 8-bit weights: half a step
    of e4m3 of every input, a share of the scale below 2^-6 of it, and the
    product's own bound with bf16's half step."""
    cfg = net.config
    T = core.shape[0]
    normed = f8.rms_norm_gated(core.reshape(T, cfg.num_v_heads, cfg.head_v_dim).cpu(),
                               z.reshape(T, cfg.num_v_heads, cfg.head_v_dim).cpu(), net.norm.weight.cpu(), net.norm.eps)
    w = f8.dequantize(*_host(net.out_proj_weight))
    want = normed @ w.t()
    scales = f8.spread(f8.block_scales(normed), *normed.shape)
    off = normed.abs() * (f8.HALF_STEP + 3 * DELTA) + 1.001 * scales * f8.HALF_STEP_SUBNORMAL
    one = torch.ones(T, -(-normed.shape[1] // 128), dtype=torch.float64)
    loss = f8.linear_bound(normed.abs() + off, one, w, one[:1].expand(w.shape[0], -1)) + off @ w.abs().t()
    err = (y.cpu().double() - want).abs()
    assert (err <= loss + 2.0 ** -8 * (want.abs() + loss)).all(), float((err / loss).max())


def test_prefill_then_decode_with_8_bit_projections():
    from logssms_amd.cache import LinearStatePool
    from logssms_amd.core import Batch, Context, Request, clear_global_ctx, set_global_ctx
    from logssms_amd.kernel import Fp8Tensor
    from logssms_amd.layers import RMSNorm
    g = gen(290)
    hidden, H, HV, dk, dv, layer_idx = 192, 2, 4, 64, 64, 1
    net = _layer(g, hidden, H, HV, dk, dv, layer_idx)
    net.quantize_weights()
    assert isinstance(net.in_proj_qkvz_weight, Fp8Tensor) and isinstance(net.out_proj_weight, Fp8Tensor)
    assert net.in_proj_ba_weight.dtype == torch.bfloat16
    cfg = net.config
    front = RMSNorm(hidden, 1e-6, weight_offset=1.0)
    front.weight = randn(hidden, g=g, std=0.2).to(DEV)
    page, slots = 64, 48
    pool = LinearStatePool(slots, 2, cfg.conv_dim, 4, HV, dk, dv, DEV, torch.bfloat16)
    pool.conv_state.copy_(randn(*pool.conv_state.shape, g=g, dtype=torch.bfloat16))
    pool.recurrent_state.copy_(randn(*pool.recurrent_state.shape, g=g, std=0.1))
    perm = torch.randperm(slots, generator=g).tolist()
    table = [[perm[(6 * i + p // page) % slots] for p in range(384)] for i in range(3)]
    reqs = [(0, 0, 70), (1, 128, 200), (2, 64, 129)]  # (table row, cached, device_len)
    T = sum(e - c for _, c, e in reqs)
    ctx = Context(page_size=page, linear_state=pool, state_table=torch.tensor(table, device=DEV))
    set_global_ctx(ctx)
    try:
        conv_ref, state_ref = pool.conv_state.cpu(), pool.recurrent_state.cpu()
        for phase in ("prefill", "decode"):
            n = T if phase == "prefill" else len(reqs)
            x, res = (randn(n, hidden, g=g, dtype=torch.bfloat16).to(DEV) for _ in range(2))
            if phase == "prefill":
                batch = Batch(reqs=[Request(t, c, e) for t, c, e in reqs], phase="prefill")
            else:
                batch = Batch(reqs=[Request(t, e, e + 1) for t, _, e in reqs], phase="decode")
            ctx.batch = batch
            ctx.linear_attn_backend.prepare_metadata(batch)
            q, y, total = front.forward_fp8(x, res)
            _, want = f8.rms_norm(x.cpu(), front.weight.cpu(), 1e-6, residual=res.cpu(), weight_offset=1.0)
            assert_quantised(q, want)
            mixed, z, beta, gate = net.proj(y, q)
            check(torch.cat([mixed, z], 1), _host(q), _host(net.in_proj_qkvz_weight), torch.bfloat16)
            assert torch.equal(torch.cat([beta, gate], 1), torch.nn.functional.linear(y, net.in_proj_ba_weight))
            if phase == "prefill":
                meta = md.prefill_metadata(table, [(t, c, e - c) for t, c, e in reqs], page)
                cu = md.from_lengths([e - c for _, c, e in reqs])["cu_seqlens"]
                core = ref.forward_prefill(mixed.cpu(), gate.cpu(), beta.cpu(), net.conv1d_weight.cpu(),
                                           net.A_log.cpu(), net.dt_bias.cpu(), conv_ref, state_ref, layer_idx,
                                           torch.tensor(cu), meta["baseline_slots"], meta["chunk_write_slots"],
                                           meta["conv_token_slots"], H, dk, HV, dv)
            else:
                read, write = md.decode_slots(table, [(t, e) for t, _, e in reqs])
                core = ref.forward_decode(mixed.cpu(), gate.cpu(), beta.cpu(), net.conv1d_weight.cpu(),
                                          net.A_log.cpu(), net.dt_bias.cpu(), conv_ref, state_ref, layer_idx,
                                          torch.tensor(read), torch.tensor(write), H, dk, HV, dv)
            start = pool.conv_state.clone(), pool.recurrent_state.clone()
            got_core = net.attend(mixed, beta, gate)
            torch.testing.assert_close(got_core.float().cpu().reshape(n, -1), core.float().reshape(n, -1), rtol=2e-2,
                                       atol=1e-2)
            torch.testing.assert_close(pool.conv_state.cpu(), conv_ref, rtol=0, atol=0)
            assert_state_close(pool.recurrent_state, state_ref)
            staged = net.output(got_core, z)
            _check_output(net, got_core, z, staged)
            # the whole call, from the same pools, is the stages one after the other
            pool.conv_state.copy_(start[0])
            pool.recurrent_state.copy_(start[1])
            assert torch.equal(net.forward(y, q), staged)
            # without the norm's rows the layer quantises its input itself
            pool.conv_state.copy_(start[0])
            pool.recurrent_state.copy_(start[1])
            own = net.forward(y)
            assert own.shape == (n, hidden) and own.isfinite().all()
            state_ref = pool.recurrent_state.cpu()
            conv_ref = pool.conv_state.cpu()
    finally:
        clear_global_ctx()


def test_weights_may_be_a_checkpoints_blocks():
    """Values and scales set from outside, the second projection alone in 8 bits."""
    from logssms_amd.kernel import Fp8Tensor, quantize_fp8_weight
    from logssms_amd.layers import GatedDeltaNet
    net = GatedDeltaNet(64, 2, 4, 32, 32, 4, 1e-6, 0, device=DEV, dtype=torch.bfloat16)
    g = gen(7)
    w = randn(64, 128, g=g, std=0.1)
    values, scales = quantize_fp8_weight(w)
    net.out_proj_weight = Fp8Tensor(values.to(DEV), scales.to(DEV))
    core = randn(9, 4, 32, g=g, dtype=torch.bfloat16).to(DEV)
    z = randn(9, 4 * 32, g=g, dtype=torch.bfloat16).to(DEV)
    _check_output(net, core, z, net.output(core, z))
    with pytest.raises(AssertionError):
        net.proj(torch.zeros(3, 64, device=DEV, dtype=torch.bfloat16), Fp8Tensor(values, scales))
    net.quantize_weights()
    assert isinstance(net.in_proj_qkvz_weight, Fp8Tensor) and net.out_proj_weight.values.data_ptr() != 0


def test_decode_step_replays():
    """The layer's decode in a graph: norm, projections, backend, gated norm,
    output; replayed on new inputs and pools beside eager calls."""
    from logssms_amd.kernel.linear_attention.fused_backend import decode_step
    from logssms_amd.layers import RMSNorm
    g = gen(291)
    hidden, H, HV, d, B = 128, 2, 4, 64, 5
    net = _layer(g, hidden, H, HV, d, d, 0)
    net.quantize_weights()
    cfg = net.config
    front = RMSNorm(hidden, 1e-6)
    front.weight = front.weight.to(DEV)
    x, res = (randn(B, hidden, g=g, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    conv0 = randn(16, 1, cfg.conv_dim, 3, g=g, dtype=torch.bfloat16).to(DEV)
    state0 = randn(16, 1, HV, d, d, g=g, std=0.1).to(DEV)
    conv, state = conv0.clone(), state0.clone()
    reads, writes = torch.arange(B, device=DEV), torch.arange(B, 2 * B, device=DEV)

    def call():
        q, y, total = front.forward_fp8(x, res)
        mixed, z, beta, gate = net.proj(y, q)
        core = decode_step(mixed, gate, beta, net.conv1d_weight, net.A_log, net.dt_bias, cfg, conv, state, reads, writes)
        return net.output(core, z), total

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed = call()
    for _ in range(3):
        x.copy_(randn(B, hidden, g=g, dtype=torch.bfloat16).to(DEV))
        conv.copy_(conv0)
        state.copy_(state0)
        eager = [t.clone() for t in call()]
        after = conv.clone(), state.clone()
        conv.copy_(conv0)
        state.copy_(state0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphed, eager))
        assert torch.equal(conv, after[0]) and torch.equal(state, after[1])
