"""Rotary positions, cache appends and paged attention on the CPU: the
frequencies of each scaling, the oracle against torch's own operators, the pool's
cache views, and every refusal that is made before a launch."""

import math
import os

import pytest
import torch

from oracle import attention as ref


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _built():
    from logssms_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.lib()


# ------------------------------------------------------------------ frequencies

def test_plain_and_stretched_frequencies():
    from logssms_amd.kernel import rotary_embedding
    plain = rotary_embedding(64, 1e4)
    want = [1e4 ** (-2 * i / 64) / (2 * math.pi) for i in range(32)]
    assert plain.turns.dtype == torch.float64 and plain.rotated == 64 and plain.scale == 1.0
    torch.testing.assert_close(plain.turns, torch.tensor(want, dtype=torch.float64), rtol=1e-14, atol=0)
    torch.testing.assert_close(rotary_embedding(64, 1e4, scaling="linear", factor=4.0).turns, plain.turns / 4, rtol=1e-14,
                               atol=0)
    base = rotary_embedding(64, 1e4, scaling="base", factor=8.0).turns
    assert base[0] == plain.turns[0]
    torch.testing.assert_close(base[-1], plain.turns[-1] / 8, rtol=1e-12, atol=0)
    # by wavelength: untouched above four rotations over the old length, divided below one, between in between
    got = rotary_embedding(64, 1e4, scaling="wavelength", factor=8.0, original_length=2048).turns
    rotations = 2048 * plain.turns
    assert torch.equal(got[rotations >= 4], plain.turns[rotations >= 4])
    torch.testing.assert_close(got[rotations <= 1], plain.turns[rotations <= 1] / 8, rtol=1e-14, atol=0)
    middle = (rotations > 1) & (rotations < 4)
    assert middle.any() and (got[middle] < plain.turns[middle]).all() and (got[middle] > plain.turns[middle] / 8).all()
    # the ramp over the pairs: monotone between both ends, and the values' scale
    yarn = rotary_embedding(64, 1e4, scaling="yarn", factor=8.0, original_length=2048)
    ratio = plain.turns / yarn.turns
    assert ratio[0] == 1.0 and ratio[-1] == pytest.approx(8.0) and (ratio.diff() >= -1e-12).all()
    assert yarn.scale == pytest.approx(0.1 * math.log(8.0) + 1.0)
    assert rotary_embedding(64, scaling="yarn", factor=8.0, original_length=2048, scale=1.0).scale == 1.0
    assert rotary_embedding(0).rotated == 0 and rotary_embedding(2, scaling="base", factor=2.0).rotated == 2


@pytest.mark.parametrize("bad", [
    dict(rotated=63), dict(rotated=-2), dict(rotated=64, base=0.0), dict(rotated=64, factor=0.0, scaling="linear"),
    dict(rotated=64, scaling="other"), dict(rotated=64, scaling="yarn", factor=2.0), dict(rotated=64, factor=2.0),
    dict(rotated=64, scaling="wavelength", factor=2.0, original_length=100, slow=4.0, fast=4.0)])
def test_frequencies_refused(bad):
    from logssms_amd.kernel import rotary_embedding
    with pytest.raises(AssertionError):
        rotary_embedding(**bad)


# ------------------------------------------------------------------ the oracle

@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation_by_complex_numbers(interleaved):
    x = torch.randn(5, 3, 16, generator=_gen(1), dtype=torch.float64)
    turns = torch.rand(4, generator=_gen(2), dtype=torch.float64)
    pos = torch.tensor([0, 1, 7, 100000, 2 ** 31 - 1])
    y = ref.rotary(x, pos, turns, interleaved, 1.5)
    unit = 1.5 * torch.polar(torch.ones(5, 4, dtype=torch.float64), 2 * math.pi * torch.remainder(pos[:, None] * turns, 1))
    part = x[..., :8]
    z = torch.complex(part[..., 0::2], part[..., 1::2]) if interleaved else torch.complex(part[..., :4], part[..., 4:])
    z = z * unit[:, None]
    got = torch.complex(y[..., 0:8:2], y[..., 1:8:2]) if interleaved else torch.complex(y[..., :4], y[..., 4:8])
    torch.testing.assert_close(got, z, rtol=1e-9, atol=1e-9)
    assert torch.equal(y[..., 8:], x[..., 8:])


def test_oracle_attention_against_torch():
    g = _gen(3)
    k_cache, v_cache = torch.randn(2, 6, 16, 2, 64, generator=g).unbind(0)
    q = torch.randn(9, 4, 64, generator=g)
    table, lens, cu = torch.tensor([[3, 1, 5], [0, 7, 2], [4, 4, 4]]), torch.tensor([40, 37, 0]), torch.tensor([0, 5, 8, 9])
    out, lse, _, _ = ref.attention(q, k_cache, v_cache, table, lens, cu, 0.125)
    for r, (a, b) in enumerate([(0, 5), (5, 8)]):
        n, count = int(lens[r]), b - a
        k = torch.cat([k_cache[p] if p < 6 else torch.zeros(16, 2, 64) for p in table[r].tolist()])[:n].double()
        v = torch.cat([v_cache[p] if p < 6 else torch.zeros(16, 2, 64) for p in table[r].tolist()])[:n].double()
        mask = torch.ones(count, n, dtype=torch.bool).tril(n - count)
        want = torch.nn.functional.scaled_dot_product_attention(
            q[a:b].double().transpose(0, 1), k.transpose(0, 1).repeat_interleave(2, 0),
            v.transpose(0, 1).repeat_interleave(2, 0), attn_mask=mask, scale=0.125).transpose(0, 1)
        torch.testing.assert_close(out[a:b], want)
    assert (out[8] == 0).all() and (lse[8] == -math.inf).all()


# ------------------------------------------------------------------ the pool's views

def test_pool_blocks_as_caches():
    from types import SimpleNamespace

    from logssms_amd.cache import HybridBlockLayout, HybridBlockPool
    spec = SimpleNamespace(num_layers=3, state_shape=(2, 32, 32), conv_shape=(128, 3))
    layout = HybridBlockLayout.make(2, spec, kv_heads=2, head_dim=64, block_size=64)
    pool = HybridBlockPool(layout, 9, "cpu", torch.bfloat16)
    slot = pool.allocate_state()
    pool.recurrent_state[pool._starts(slot)[0], 1] = 3.0
    block = pool.allocator.take_run(1)
    k, v = pool.kv_cache(1)
    assert k.shape == v.shape == (9, 64, 2, 64) and k.stride(3) == 1
    before = pool.storage.clone()
    k[block], v[block] = 1.0, 2.0
    changed = pool.storage != before
    assert changed[1, block].all() and int(changed.sum()) == layout.layer_elements
    assert (pool.storage[1, block, :64 * 128] == 1).all() and (pool.storage[1, block, 64 * 128:] == 2).all()


# ------------------------------------------------------------------ refusals

def test_rotary_refuses_what_does_not_fit():
    from logssms_amd.kernel import Rotary, apply_rotary, rotary_embedding
    _built()
    q, k, pos, rot = torch.zeros(4, 3, 32), torch.zeros(4, 1, 32), torch.arange(4), rotary_embedding(16)
    for bad in (
        lambda: apply_rotary(q[0], None, pos, rot),
        lambda: apply_rotary(q, k[:3], pos, rot),
        lambda: apply_rotary(q, k[..., :16], pos, rot),
        lambda: apply_rotary(q, k.bfloat16(), pos, rot),
        lambda: apply_rotary(q, k, pos[:3], rot),
        lambda: apply_rotary(q, k, pos[None], rot),
        lambda: apply_rotary(q, k, pos, rotary_embedding(34)),  # more than the head has
        lambda: apply_rotary(q, k, pos, Rotary(rot.turns.float())),
        lambda: apply_rotary(q, k, pos, Rotary(rot.turns[None])),
        lambda: apply_rotary(q, None, pos, rot, k_out=k),
        lambda: apply_rotary(q, k, pos, rot, q_out=k),
        lambda: apply_rotary(q, k, pos, rot, q_out=q.bfloat16()),
        lambda: apply_rotary(q, k, pos, rot, q_out=torch.zeros(1, 3, 32).expand(4, 3, 32)),
        lambda: apply_rotary(q, k, pos, rot, q_out=torch.zeros(4, 3, 64)[..., ::2]),
        lambda: apply_rotary(q, k, pos, rot, q_out=torch.zeros(4 * 3 * 32).as_strided((4, 3, 32), (32, 16, 1))),
    ):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: apply_rotary(q, k, pos.float(), rot), lambda: apply_rotary(q.double(), k.double(), pos, rot),
                lambda: apply_rotary(3, k, pos, rot)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="ROCm"):
        apply_rotary(q, k, pos, rot)


def test_append_refuses_what_does_not_fit():
    from logssms_amd.kernel import append_paged_kv, rotary_embedding
    _built()
    k, cache, slots, rot = torch.zeros(4, 2, 32), torch.zeros(5, 8, 2, 32), torch.arange(4), rotary_embedding(16)
    q = torch.zeros(4, 6, 32)
    ok = dict(positions=slots, rotary=rot, q=q)
    for bad in (
        lambda: append_paged_kv(k[0], k[0], cache, cache, slots),
        lambda: append_paged_kv(k, k[:, :1], cache, cache, slots),
        lambda: append_paged_kv(k, k.half(), cache, cache, slots),
        lambda: append_paged_kv(k, k, cache.half(), cache, slots),
        lambda: append_paged_kv(k, k, cache[:, :, :1], cache, slots),
        lambda: append_paged_kv(k, k, cache[0], cache, slots),
        lambda: append_paged_kv(k, k, cache, cache[:4], slots),
        lambda: append_paged_kv(k, k, cache, torch.zeros(5, 8, 2, 64)[..., ::2], slots),
        lambda: append_paged_kv(k, k, cache, cache, slots[:3]),
        lambda: append_paged_kv(k, k, cache, cache, slots, positions=slots),  # without a rotation
        lambda: append_paged_kv(k, k, cache, cache, slots, rotary=rot),  # without positions
        lambda: append_paged_kv(k, k, cache, cache, slots, positions=slots[:2], rotary=rot),
        lambda: append_paged_kv(k, k, cache, cache, slots, **{**ok, "q": q[:3]}),
        lambda: append_paged_kv(k, k, cache, cache, slots, **{**ok, "q": q.half()}),
        lambda: append_paged_kv(k, k, cache, cache, slots, q_out=q),
        lambda: append_paged_kv(k, k, cache, cache, slots, **ok, q_out=q[:, :2]),
    ):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        append_paged_kv(k, k, cache, cache, slots.float())
    with pytest.raises(RuntimeError, match="ROCm"):
        append_paged_kv(k, k, cache, cache, slots, **ok)


def test_attention_refuses_what_does_not_fit():
    from logssms_amd.kernel import paged_attention
    _built()
    q = torch.zeros(3, 4, 64).bfloat16()
    cache = torch.zeros(5, 16, 2, 64).bfloat16()
    table, lens, shared = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.tensor([16])
    ok = (q, cache, cache, table, lens)

    def call(*args, **kw):
        return lambda: paged_attention(*args, **kw)
    for bad in (
        call(q[0], *ok[1:]), call(q.float(), cache.float(), cache.float(), table, lens),
        call(q, cache.half(), cache, table, lens), call(q, cache[0], cache, table, lens),
        call(q, cache, cache[:4], table, lens), call(q[:, :3], *ok[1:]),  # 3 heads on 2
        call(q, torch.zeros(5, 16, 2, 32).bfloat16(), cache, table, lens),
        call(q, cache, cache, table[0], lens), call(q, cache, cache, table, lens[:2]),
        call(q[:2], cache, cache, table, lens),  # a token each, without cu_seqlens
        call(*ok, cu_seqlens=torch.arange(3)), call(*ok, group_offsets=torch.tensor([0, 3])),
        call(*ok, shared_lens=shared[:0]), call(*ok, shared_lens=torch.tensor([16, 16])),  # groups of unknown extent
        call(*ok, shared_lens=shared, group_offsets=torch.tensor([0, 1, 3])),
        call(*ok, out=torch.zeros(3, 4, 64)), call(*ok, out=q[:2]), call(*ok, out=q[:1].expand(3, 4, 64)),
    ):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        paged_attention(q, cache, cache, table.float(), lens)
    with pytest.raises(TypeError):
        paged_attention(q, cache, cache, table, lens, shared_lens=shared.float())
    with pytest.raises(RuntimeError, match="ROCm"):
        paged_attention(*ok)


def _attend(lib, **kw):
    """gdn_paged_attention with dummy addresses that are never read: only what is
    refused before a launch is called through this."""
    a = dict(q=0x10000, q_token=256, q_head=64, dtype=1, tokens=3, heads=4, dim=64, k=0x10000, k_page=2048, k_token=128,
             k_head=64, v=0x10000, v_page=2048, v_token=128, v_head=64, kv_heads=2, pages=5, page=16, table=0x10000,
             table_dtype=0, table_row=2, width=2, lens=0x10000, lens_dtype=0, requests=3, shared=None, shared_dtype=0,
             offsets=None, offsets_dtype=0, groups=0, cu=None, cu_dtype=0, scale=0.125, out=0x10000, out_token=256,
             out_head=64, lse=None, ws=0x10000, ws_bytes=0, stream=None)
    a.update(kw)
    return lib.gdn_paged_attention(*a.values())


def test_c_entries_refuse_without_launching():
    lib = _built()
    for kw in (dict(dtype=0), dict(heads=3), dict(page=24), dict(page=0), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=math.inf), dict(scale=math.nan), dict(tokens=4), dict(groups=1), dict(groups=2, shared=0x10000),
               dict(q=0x10008), dict(k=0x10008), dict(q_token=252), dict(v_page=2044), dict(k_token=-128),
               dict(k_token=1 << 24), dict(out=0x10004), dict(out_head=62), dict(table_dtype=3), dict(lens=None),
               dict(ws=None), dict()):  # the last: no room in the workspace
        assert _attend(lib, **kw) == 1, kw
        assert lib.gdn_last_error()
    for kw in (dict(dim=96), dict(width=1 << 28), dict(tokens=1 << 30, requests=1 << 30)):
        assert _attend(lib, **kw) == 2, kw
    assert _attend(lib, tokens=0, requests=0) == 0  # nothing to do
    assert _attend(lib, tokens=3, requests=0, cu=0x10000) == 0
    d = 0x10000
    turn = lambda **kw: lib.gdn_apply_rotary(*{**dict(  # noqa: E731
        q=d, qt=64, qh=32, heads=2, k=None, kt=0, kh=0, k_heads=0, dtype=1, tokens=3, dim=32, pos=d, pd=0, turns=d,
        rotated=16, inter=0, scale=1.0, qo=d, qot=64, qoh=32, ko=None, kot=0, koh=0, stream=None), **kw}.values())
    for kw in (dict(dtype=5), dict(rotated=15), dict(rotated=34), dict(rotated=-2), dict(pos=None), dict(turns=None),
               dict(pd=7), dict(q=None), dict(qo=None), dict(k_heads=1), dict(heads=-1), dict(dim=0)):
        assert turn(**kw) == 1, kw
    assert turn(heads=1 << 20) == 2 and turn(dim=8192, rotated=0) == 2
    assert turn(tokens=0, q=None) == 0 and turn(heads=0) == 0
    assert lib.gdn_paged_attention_workspace_bytes(0, 3, 0, 4, 2, 64, 0) == 0
    assert lib.gdn_paged_attention_workspace_bytes(3, 3, 0, 4, 2, 64, 0) > 0


def test_append_refuses_caches_on_top_of_themselves():
    from logssms_amd.kernel import append_paged_kv
    _built()
    k, cache, slots = torch.zeros(4, 2, 32), torch.zeros(5, 8, 2, 32), torch.arange(4)
    for view in (cache[:1].expand(5, 8, 2, 32), cache[:, :1].expand(5, 8, 2, 32), cache[:, :, :1].expand(5, 8, 2, 32),
                 torch.zeros(5 * 8 * 2 * 32).as_strided((5, 8, 2, 32), (512, 64, 16, 1))):
        for caches in ((view, cache), (cache, view)):
            with pytest.raises(AssertionError, match="overlap"):
                append_paged_kv(k, k, *caches, slots)


def test_more_rows_than_a_launch_has_threads_for():
    lib = _built()
    assert _attend(lib, tokens=1 << 24, requests=1 << 24) == 2  # 2^26 rows
    d = 0x10000
    turn = dict(q=d, qt=64, qh=32, heads=2, k=None, kt=0, kh=0, k_heads=0, dtype=1, tokens=3, dim=32, pos=d, pd=0, turns=d,
                rotated=16, inter=0, scale=1.0, qo=d, qot=64, qoh=32, ko=None, kot=0, koh=0, stream=None)
    turn.update(dim=4096, tokens=1 << 24)
    assert lib.gdn_apply_rotary(*turn.values()) == 2


def test_the_largest_launch_that_joins_pieces():
    """A block of 256 threads joins four rows, and a launch has up to 2^32 - 1 threads."""
    lib = _built()
    one = dict(heads=1, kv_heads=1, requests=1, cu=0x10000)
    for rows in ((1 << 26) - 3, (1 << 26) - 1):
        assert _attend(lib, tokens=rows, **one) == 2, rows
    assert _attend(lib, tokens=((1 << 26) - 1) // 3, **{**one, "heads": 3}) == 2
    assert _attend(lib, tokens=(1 << 26) - 4, **one) == 1  # not its size: no room in the workspace


@pytest.mark.parametrize("strides", [
    (512, 32, 32, 1),  # a head is the next token's first
    (64, 256, 32, 1),  # pages inside tokens: the last page is the first one's next token
    (512, 512, 32, 1),  # a page's second token is the next page's first
    (480, 64, 32, 1),  # half of a page's last token is the next page's
    (64, 160, 32, 1), (32, 160, 768, 1)])
def test_append_refuses_caches_whose_axes_coincide(strides):
    """Every stride is a row or more, and rows lie on top of each other all the same."""
    from logssms_amd.kernel import append_paged_kv
    _built()
    k, cache, slots = torch.zeros(4, 2, 32), torch.zeros(5, 8, 2, 32), torch.arange(4)
    view = torch.zeros(5 * 8 * 1024).as_strided((5, 8, 2, 32), strides)
    at = torch.arange(view.untyped_storage().nbytes() // 4).as_strided(view.shape, strides)
    assert at.unique().numel() < view.numel()
    for caches in ((view, cache), (cache, view)):
        with pytest.raises(AssertionError, match="overlap"):
            append_paged_kv(k, k, *caches, slots)


@pytest.mark.parametrize("strides", [
    (1024, 64, 32, 1),  # the pool's: keys, then values
    (512, 32, 256, 1), (1024, 32, 256, 1),  # heads first
    (64, 320, 32, 1), (32, 320, 160, 1),  # pages inside tokens
    (600, 70, 33, 1)])
def test_append_takes_caches_in_any_order(strides):
    from logssms_amd.kernel import append_paged_kv
    _built()
    k, cache, slots = torch.zeros(4, 2, 32), torch.zeros(5, 8, 2, 32), torch.arange(4)
    view = torch.zeros(5 * 8 * 1024).as_strided((5, 8, 2, 32), strides)
    for caches in ((view, cache), (cache, view)):
        with pytest.raises(RuntimeError, match="ROCm"):  # no other objection
            append_paged_kv(k, k, *caches, slots)
