"""Rotary positions and cache appends on the GPU against 64 bits."""

import pytest
import torch

from gpu_util import DEV, gen, randn
from oracle import attention as ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _rotary(n, **kw):
    from logssms_amd.kernel import rotary_embedding
    return rotary_embedding(n, 1e4, **kw)


def _on(rotary):
    return rotary._replace(turns=rotary.turns.to(DEV))


def _check(got, x, positions, rotary):
    want = ref.rotary(x, positions, rotary.turns, rotary.interleaved, rotary.scale)
    bound = ref.rotary_bound(x, rotary.turns, rotary.interleaved, rotary.scale, x.dtype, want)
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), f"off by {float((err - bound).max()):.3e} more than the bound"
    rest = slice(rotary.rotated, None)
    assert torch.equal(got.cpu()[..., rest], x[..., rest])


@pytest.mark.parametrize("io", list(TYPES))
@pytest.mark.parametrize("tokens,heads,k_heads,dim,rotated,interleaved", [
    (1, 16, 2, 256, 64, False), (1, 16, 2, 256, 64, True), (37, 3, 3, 64, 64, False), (37, 3, 1, 64, 64, True),
    (9, 2, 1, 96, 24, False), (9, 2, 1, 96, 24, True), (5, 1, 0, 7, 4, False), (5, 1, 0, 7, 6, True),
    (300, 5, 2, 40, 10, False), (2, 32, 8, 128, 2, True), (3, 1, 1, 4096, 4096, False), (1025, 1, 1, 16, 16, False)])
def test_rotary_matches_64_bits(io, tokens, heads, k_heads, dim, rotated, interleaved):
    from logssms_amd.kernel import apply_rotary
    g = gen(tokens + dim)
    rotary = _rotary(rotated, interleaved=interleaved)
    q, k = (randn(tokens, n, dim, g=g, dtype=TYPES[io]) for n in (heads, k_heads))
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g)
    got = apply_rotary(q.to(DEV), k.to(DEV) if k_heads else None, positions.to(DEV), _on(rotary))
    _check(got[0], q, positions, rotary)
    if k_heads:
        _check(got[1], k, positions, rotary)
    else:
        assert got[1] is None


@pytest.mark.parametrize("scaling", ["linear", "base", "wavelength", "yarn"])
def test_far_positions_and_scalings(scaling):
    from logssms_amd.kernel import apply_rotary
    rotary = _rotary(32, scaling=scaling, factor=8.0, original_length=4096)
    positions = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 - 1, -1, -(2 ** 31)])
    q = randn(6, 2, 32, g=gen(1))
    for dtype in (torch.int32, torch.int64):
        _check(apply_rotary(q.to(DEV), None, positions.to(dtype).to(DEV), _on(rotary))[0], q, positions, rotary)


@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_views_odd_addresses_and_in_place(interleaved):
    from logssms_amd.kernel import apply_rotary
    rotary = _rotary(32, interleaved=interleaved)
    g = gen(5)
    positions = torch.arange(11)
    merged = randn(11, 9 * 64 + 3, g=g, dtype=torch.bfloat16)
    for offset in (0, 8, 3):  # rows at multiples of 16 bytes, or at odd addresses
        rows = merged[:, offset:offset + 9 * 64].reshape(11, 9, 64) if offset == 3 else None
        wide = torch.zeros(11, 9 * 64 + (16 if offset != 3 else 3), dtype=torch.bfloat16)
        wide[:, offset:offset + 9 * 64] = merged[:, :9 * 64] if rows is None else rows.view(11, -1)
        on = wide.to(DEV)
        view = on[:, offset:offset + 9 * 64].unflatten(1, (9, 64))
        q, k = view[:, :7], view[:, 7:]
        plain_q, plain_k = q.cpu().clone(), k.cpu().clone()
        got = apply_rotary(q, k, positions.to(DEV), _on(rotary))
        _check(got[0], plain_q, positions, rotary)
        _check(got[1], plain_k, positions, rotary)
        # heads first, and channels that are not side by side
        _check(apply_rotary(q.transpose(0, 1).contiguous().transpose(0, 1), None, positions.to(DEV), _on(rotary))[0],
               plain_q, positions, rotary)
        _check(apply_rotary(q.permute(0, 2, 1).contiguous().permute(0, 2, 1), None, positions.to(DEV), _on(rotary))[0],
               plain_q, positions, rotary)
        # in place, the columns around it as they were
        around = on.cpu().clone()
        out = apply_rotary(q, k, positions.to(DEV), _on(rotary), q_out=q, k_out=k)
        assert out[0].data_ptr() == q.data_ptr()
        assert torch.equal(q, got[0]) and torch.equal(k, got[1])
        assert torch.equal(on.cpu()[:, :offset], around[:, :offset])
        assert torch.equal(on.cpu()[:, offset + 9 * 64:], around[:, offset + 9 * 64:])


def test_rotary_of_nothing():
    from logssms_amd.kernel import apply_rotary
    rotary = _on(_rotary(16))
    q = torch.empty(0, 2, 32, device=DEV)
    assert apply_rotary(q, None, torch.empty(0, dtype=torch.int64, device=DEV), rotary)[0].shape == (0, 2, 32)
    q = torch.randn(3, 2, 32, device=DEV)
    none = _on(_rotary(0))
    assert torch.equal(apply_rotary(q, None, torch.arange(3, device=DEV), none)[0], q)


def test_not_finite_values_stay_in_their_pair():
    from logssms_amd.kernel import apply_rotary
    q = torch.ones(1, 2, 32)
    q[0, 0, 3], q[0, 1, 20] = float("nan"), float("inf")
    got = apply_rotary(q.to(DEV), None, torch.tensor([5], device=DEV), _on(_rotary(32)))[0].cpu()
    bad = ~got.isfinite()
    assert bad[0, 0].nonzero().flatten().tolist() == [3, 19] and bad[0, 1].nonzero().flatten().tolist() == [4, 20]


# ------------------------------------------------------------------ append

def _cache(pages, page, heads, dim, dtype, views):
    storage = torch.full((pages, 2, page, heads, dim), 7.0).to(dtype).to(DEV)
    if views:
        return storage, storage[:, 0], storage[:, 1]
    k = storage[:, 0].contiguous()
    return storage, k, storage[:, 1].contiguous()


@pytest.mark.parametrize("io", list(TYPES))
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotated,interleaved,page,views", [
    (1, 16, 2, 256, 64, False, 64, True), (33, 4, 2, 64, 64, True, 16, True), (70, 0, 3, 40, 10, False, 5, False),
    (129, 5, 1, 48, 48, False, 48, True), (20, 2, 2, 9, 0, False, 3, False), (300, 0, 1, 128, 0, False, 64, True)])
def test_append_writes_its_slots_only(io, tokens, heads, kv_heads, dim, rotated, interleaved, page, views):
    from logssms_amd.kernel import append_paged_kv
    g = gen(tokens)
    dtype = TYPES[io]
    pages = -(-2 * tokens // page) + 1
    rotary = _rotary(rotated, interleaved=interleaved)
    k, v, q = randn(tokens, kv_heads, dim, g=g, dtype=dtype), randn(tokens, kv_heads, dim, g=g, dtype=dtype), None
    if heads:
        q = randn(tokens, heads, dim, g=g, dtype=dtype)
    positions = torch.randint(0, 100000, (tokens,), generator=g)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[3], slots[4] = -1, pages * page, -(2 ** 31)  # no such slot: nothing is written
    for index in (torch.int32, torch.int64):
        storage, k_cache, v_cache = _cache(pages, page, kv_heads, dim, dtype, views)
        q_on = None if q is None else q.to(DEV)
        got = append_paged_kv(k.to(DEV), v.to(DEV), k_cache, v_cache, slots.to(index).to(DEV),
                              positions=positions.to(DEV) if rotated else None, rotary=_on(rotary) if rotated else None,
                              q=q_on)
        flat_k, flat_v = k_cache.cpu().reshape(-1, kv_heads, dim), v_cache.cpu().reshape(-1, kv_heads, dim)
        there = (slots >= 0) & (slots < pages * page)
        assert torch.equal(flat_v[slots[there]], v[there])
        _check(flat_k[slots[there]], k[there], positions[there], rotary)
        others = torch.ones(pages * page, dtype=torch.bool)
        others[slots[there]] = False
        assert (flat_k[others] == 7).all() and (flat_v[others] == 7).all()
        if heads:
            _check(got, q, positions, rotary)
            assert torch.equal(q_on.cpu(), q)
            again = append_paged_kv(k.to(DEV), v.to(DEV), k_cache, v_cache, slots.to(DEV),
                                    positions=positions.to(DEV) if rotated else None,
                                    rotary=_on(rotary) if rotated else None, q=q_on, q_out=q_on)
            assert again.data_ptr() == q_on.data_ptr() and torch.equal(q_on, got)
        else:
            assert got is None


def test_append_far_into_a_large_cache():
    """Slots whose byte offsets pass 32 bits."""
    from logssms_amd.kernel import append_paged_kv
    pages, page, heads, dim = 5000, 256, 8, 256
    storage = torch.empty(pages, 2, page, heads, dim, dtype=torch.bfloat16, device=DEV)  # 10 GB
    k_cache, v_cache = storage[:, 0], storage[:, 1]
    slots = torch.tensor([0, pages * page - 1, 600000, 1200001])
    k, v = randn(2, 4, heads, dim, g=gen(9), dtype=torch.bfloat16).unbind(0)
    append_paged_kv(k.to(DEV), v.to(DEV), k_cache, v_cache, slots.to(DEV))
    assert torch.equal(k_cache[slots.to(DEV) // page, slots.to(DEV) % page].cpu(), k)
    assert torch.equal(v_cache[slots.to(DEV) // page, slots.to(DEV) % page].cpu(), v)


def test_append_in_a_graph_follows_its_slots():
    from logssms_amd.kernel import append_paged_kv
    rotary = _on(_rotary(32))
    k, v = (torch.randn(6, 2, 64, device=DEV).bfloat16() for _ in range(2))
    slots, positions = torch.arange(6, device=DEV), torch.arange(6, device=DEV)
    _, k_cache, v_cache = _cache(8, 16, 2, 64, torch.bfloat16, True)
    append_paged_kv(k, v, k_cache, v_cache, slots, positions=positions, rotary=rotary, q=k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = append_paged_kv(k, v, k_cache, v_cache, slots, positions=positions, rotary=rotary, q=k)
    for i in range(1, 4):
        slots.copy_(torch.randperm(128)[:6])
        positions.add_(1000 * i)
        k_cache.zero_()
        v_cache.zero_()
        graph.replay()
        got = k_cache.clone(), v_cache.clone(), q.clone()
        k_cache.zero_()
        v_cache.zero_()
        want_q = append_paged_kv(k, v, k_cache, v_cache, slots, positions=positions, rotary=rotary, q=k)
        assert torch.equal(got[0], k_cache) and torch.equal(got[1], v_cache) and torch.equal(got[2], want_q)
        torch.cuda.synchronize()


def test_positions_and_slots_past_32_bits():
    """Whose low halves would be others."""
    from logssms_amd.kernel import append_paged_kv
    rotary = _rotary(32)
    positions = torch.tensor([2 ** 32 + 3, 2 ** 40 + 1, -(2 ** 33), 2 ** 31, 7])
    slots = torch.tensor([2 ** 32 + 1, 3, -(2 ** 33) + 2, 2 ** 40, 0])
    k, v, q = randn(3, 5, 2, 64, g=gen(11), dtype=torch.bfloat16).unbind(0)
    _, k_cache, v_cache = _cache(4, 16, 2, 64, torch.bfloat16, True)
    got = append_paged_kv(k.to(DEV), v.to(DEV), k_cache, v_cache, slots.to(DEV), positions=positions.to(DEV),
                          rotary=_on(rotary), q=q.to(DEV))
    _check(got, q, positions, rotary)
    flat_k, flat_v = k_cache.cpu().reshape(-1, 2, 64), v_cache.cpu().reshape(-1, 2, 64)
    _check(flat_k[[3, 0]], k[[1, 4]], positions[[1, 4]], rotary)
    assert torch.equal(flat_v[[3, 0]], v[[1, 4]])
    others = torch.ones(64, dtype=torch.bool)
    others[[3, 0]] = False
    assert (flat_k[others] == 7).all() and (flat_v[others] == 7).all()


def _two(storage, k_at, v_at, k_strides, v_strides, shape=(5, 8, 2, 32)):
    return storage.as_strided(shape, k_strides, k_at), storage.as_strided(shape, v_strides, v_at)


@pytest.mark.parametrize("k_at,v_at,k_strides,v_strides", [
    (0, 0, (512, 64, 32, 1), (512, 64, 32, 1)),  # the same tensor twice
    (0, 512, (512, 64, 32, 1), (512, 64, 32, 1)),  # a page further on
    (0, 2560 - 32, (512, 64, 32, 1), (512, 64, 32, 1)),  # the last head of the one, the first of the other
    (0, 480, (1024, 64, 32, 1), (1024, 64, 32, 1)),  # a page's values from its last key on
    (0, 544, (1024, 64, 32, 1), (1024, 64, 32, 1)),  # its last value the next page's first key
    (0, 16, (1024, 128, 64, 1), (1024, 128, 64, 1)),  # by heads, from half a row on
    (0, 64, (1024, 64, 512, 1), (1024, 64, 512, 1)),  # heads first, a token further on
    (0, 512, (2048, 128, 32, 1), (2048, 64, 32, 1))])  # layouts of their own, in one block
def test_caches_on_top_of_each_other_are_refused(k_at, v_at, k_strides, v_strides):
    from logssms_amd.kernel import append_paged_kv
    k_cache, v_cache = _two(torch.zeros(20000, device=DEV), k_at, v_at, k_strides, v_strides)
    held = torch.arange(20000)
    a, b = _two(held, k_at, v_at, k_strides, v_strides)
    assert torch.isin(a, b).any()
    k, slots = torch.ones(4, 2, 32, device=DEV), torch.arange(4, device=DEV)
    for caches in ((k_cache, v_cache), (v_cache, k_cache)):
        with pytest.raises(AssertionError, match="overlap"):
            append_paged_kv(k, k, *caches, slots)


@pytest.mark.parametrize("k_at,v_at,k_strides,v_strides", [
    (0, 512, (1024, 64, 32, 1), (1024, 64, 32, 1)),  # the pool's
    (0, 64, (1024, 128, 32, 1), (1024, 128, 32, 1)), (0, 32, (1024, 128, 64, 1), (1024, 128, 64, 1)),  # by tokens, by heads
    (512, 0, (1024, 32, 256, 1), (1024, 32, 256, 1)),  # heads first, values in front
    (0, 512, (1024, 64, 32, 1), (1024, 32, 256, 1)),  # keys by tokens, values by heads
    (0, 3000, (512, 64, 32, 1), (600, 70, 33, 1)),  # one behind the other
    (0, 320, (32, 640, 160, 1), (32, 640, 160, 1)),  # pages inside tokens and heads
    (0, 5 * 512 + 7, (512, 64, 32, 1), (512, 32, 256, 1))])
def test_caches_beside_each_other(k_at, v_at, k_strides, v_strides):
    """Layouts of their own, in one storage: each takes its rows, and nothing else changes."""
    from logssms_amd.kernel import append_paged_kv
    rotary = _rotary(16)
    storage = torch.full((20000,), 7.0, device=DEV)
    k_cache, v_cache = _two(storage, k_at, v_at, k_strides, v_strides)
    k, v = randn(2, 6, 2, 32, g=gen(21)).unbind(0)
    positions, slots = torch.arange(6) * 1000, torch.tensor([39, 0, 17, -1, 8, 40])
    append_paged_kv(k.to(DEV), v.to(DEV), k_cache, v_cache, slots.to(DEV), positions=positions.to(DEV),
                    rotary=_on(rotary))
    there = [0, 1, 2, 4]
    at = slots[there]
    _check(k_cache[at // 8, at % 8].cpu(), k[there], positions[there], rotary)
    assert torch.equal(v_cache[at // 8, at % 8].cpu(), v[there])
    a, b = _two(torch.arange(20000), k_at, v_at, k_strides, v_strides)
    others = torch.ones(20000, dtype=torch.bool)
    others[torch.cat([a[at // 8, at % 8], b[at // 8, at % 8]]).flatten()] = False
    assert (storage.cpu()[others] == 7).all()
