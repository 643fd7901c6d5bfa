"""Paged attention with shared prefixes on the GPU against 64 bits: head layouts,
page sizes, lengths from none to several ranges of keys, drafted and prompt tokens,
groups, empty rows, what lies in masked places, strides, graphs and streams."""

import math

import pytest
import torch

from gpu_util import DEV, gen, randn
from oracle import attention as ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


class Batch:
    """Requests of `new` tokens and `lens` positions, the first shared[g] of which lie in the pages of
    the group's first request; pages in random order, what no request owns not finite."""

    def __init__(self, seed, heads, kv_heads, dim, page, lens, new=None, shared=None, groups=None, io="bf16",
                 q_std=1.5, width=None):
        g = gen(seed)
        self.io, self.page, self.lens = TYPES[io], page, list(lens)
        n = len(lens)
        self.new = [1] * n if new is None else list(new)
        self.cu = None if new is None else torch.tensor([0] + self.new).cumsum(0)
        tokens = sum(self.new)
        self.shared = None if shared is None else torch.tensor(shared)
        self.groups = None if groups is None else torch.tensor(groups)
        need = [-(-max(0, length) // page) for length in lens]
        self.width = max(need + [1]) if width is None else width
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((n, self.width), -1)
        for r in range(n):
            first, common = r, 0
            if shared is not None:
                bounds = [0, n] if groups is None else groups
                for j in range(len(shared)):
                    if bounds[j] <= r < bounds[j + 1]:
                        first, common = bounds[j], -(-shared[j] // page)
            for p in range(min(need[r], self.width)):
                if p < common and r != first and self.table[first, p] >= 0:
                    self.table[r, p] = self.table[first, p]
                else:
                    self.table[r, p] = order.pop()
        self.k, self.v = (randn(pages, page, kv_heads, dim, g=g).to(self.io) for _ in range(2))
        self.q = randn(tokens, heads, dim, g=g, std=q_std).to(self.io)
        # everything behind the sequences' ends, and the pages of nobody
        owned = torch.zeros(pages, page, dtype=torch.bool)
        for r in range(n):
            for p in range(min(max(0, lens[r]), self.width * page)):
                owned[self.table[r, p // page], p % page] = True
        self.k[~owned], self.v[~owned] = math.nan, math.inf

    def caches(self, views=True):
        if not views:
            return self.k.to(DEV), self.v.to(DEV)
        storage = torch.stack([self.k, self.v], 1).to(DEV)
        return storage[:, 0], storage[:, 1]

    def run(self, *, index=torch.int32, scale=None, views=True, **kw):
        from logssms_amd.kernel import paged_attention
        on = lambda t: None if t is None else t.to(index).to(DEV)  # noqa: E731
        k, v = self.caches(views)
        return paged_attention(kw.pop("q", self.q.to(DEV)), k, v, on(self.table), on(torch.tensor(self.lens)),
                               shared_lens=on(self.shared), group_offsets=on(self.groups), cu_seqlens=on(self.cu),
                               scale=scale, **kw)

    def check(self, out, lse=None, scale=None):
        scale = self.q.shape[-1] ** -0.5 if scale is None else scale
        want, want_lse, bound, lse_bound = ref.attention(self.q, self.k, self.v, self.table, self.lens, self.cu, scale)
        err = (out.double().cpu() - want).abs()
        limit = ref.attention_bound(want, bound, self.io)
        bad = ~(err <= limit)
        assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                               f"{float(err[bad][0]):.3e} > {float(limit[bad][0]):.3e}")
        if lse is not None:
            got = lse.double().cpu()
            none = want_lse == -math.inf
            assert torch.equal(got == -math.inf, none)
            assert ((got - want_lse).abs()[~none] <= lse_bound[~none]).all()


LENGTHS = [1, 16, 17, 0, 31, 63, 64, 65, 128, 129, 200, 300]


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (16, 2, 256, 64), (8, 8, 64, 16), (8, 2, 128, 48), (7, 1, 64, 32), (3, 3, 256, 16), (40, 1, 128, 64), (33, 1, 256, 16)])
def test_single_tokens(io, heads, kv_heads, dim, page):
    """A token each: more than 32 heads to a key head too."""
    b = Batch(heads + dim, heads, kv_heads, dim, page, LENGTHS, io=io)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("length", [1, 2, 500, 4097])
def test_one_request(length):
    """Its keys over many blocks, to be joined."""
    b = Batch(length, 16, 2, 256, 64, [length])
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(16, 2, 256, 64), (8, 8, 64, 16), (12, 3, 128, 48)])
@pytest.mark.parametrize("shared", [16, 100, 160])
def test_single_tokens_behind_a_shared_prefix(io, heads, kv_heads, dim, page, shared):
    """Few and many rows behind it; it may end inside a page, that then is shared as well."""
    for requests in (2, 19):
        lens = [shared + (7 * r) % 60 + 1 for r in range(requests)]
        lens = [n if shared % page == 0 else shared for n in lens]  # own positions only in own pages
        b = Batch(shared + requests, heads, kv_heads, dim, page, lens, shared=[shared], io=io)
        out, lse = b.run(return_lse=True)
        b.check(out, lse)


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (8, 8, 64), (8, 2, 128), (6, 1, 128)])
def test_a_shared_length_inside_shared_pages(heads, kv_heads, dim):
    """Positions counted as shared may be fewer than those that lie in shared pages."""
    lens = [64 * 5 + 9 * r for r in range(14)]
    b = Batch(3, heads, kv_heads, dim, 64, lens, shared=[64 * 5])
    for fewer in (0, 1, 15, 33, 100, 319, 320):
        b.shared = torch.tensor([fewer])
        out, lse = b.run(return_lse=True)
        b.check(out, lse)


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(16, 2, 256, 64), (4, 4, 64, 16), (8, 2, 128, 48)])
def test_drafts_and_prompts(io, heads, kv_heads, dim, page):
    """Requests of no, one, few and many new tokens, continued or new."""
    new = [1, 5, 0, 33, 70, 8, 2]
    lens = [40, 5, 30, 90, 70, 200, 1]  # the last sees one position, its first token none
    b = Batch(heads * dim, heads, kv_heads, dim, page, lens, new=new, io=io)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_groups(index):
    """Groups of one, none and several requests with prefixes of their own, requests outside of all of
    them, lengths that end before the prefix does."""
    lens = [128 + 5, 128, 128 + 40, 64 + 1, 200 + 9, 200 + 64, 200, 30, 0]
    new = [5, 1, 9, 1, 3, 64, 2, 30, 1]
    b = Batch(8, 8, 2, 128, 8 * 16, lens, new=new, shared=[128, 0, 128, 128], groups=[0, 3, 3, 4, 7])
    # the third group's only request is shorter than its shared length, the fourth's pages are shared up to 128
    out, lse = b.run(index=index, return_lse=True)
    b.check(out, lse)


def test_padded_requests_behind_a_shared_prefix():
    """Requests that are there for their place only (length 0) and ones that end inside the shared part."""
    b = Batch(4, 16, 2, 128, 64, [128 + 20, 0, 128, 100, 0, 1, 128 + 64], shared=[128])
    out, lse = b.run(return_lse=True)
    b.check(out, lse)
    assert (out.cpu()[[1, 4]] == 0).all()


def test_tokens_of_nobody_are_left_alone():
    b = Batch(5, 4, 2, 64, 16, [40, 9, 77], new=[3, 2, 40])
    b.cu = torch.tensor([1, 4, 6, 46])
    b.q = torch.cat([b.q[:1], b.q, b.q[:3]])
    out = torch.full(b.q.shape, 5.0, dtype=b.io, device=DEV)
    got = b.run(out=out)
    assert got.data_ptr() == out.data_ptr()
    out = out.cpu()
    assert (out[0] == 5).all() and (out[46:] == 5).all()
    want, _, bound, _ = ref.attention(b.q, b.k, b.v, b.table, b.lens, b.cu, 0.125)
    assert ((out.double() - want).abs() <= ref.attention_bound(want, bound, b.io))[1:46].all()


def test_pages_outside_of_the_cache_stand_for_zeros():
    b = Batch(6, 8, 2, 128, 16, [100, 64, 200, 33], shared=[32])
    b.table[0, 3], b.table[1, 0], b.table[2, 12], b.table[2, 5] = -1, 10 ** 6, -(2 ** 31), b.k.shape[0]
    b.table[1:, :2] = b.table[0, :2]
    out, lse = b.run(return_lse=True)
    b.check(out, lse)
    b.table[0, 0] = b.k.shape[0]  # in the shared part
    b.table[1:, :2] = b.table[0, :2]
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_lengths_past_the_table():
    """What the table has no room for is not there; a token still sees by its position."""
    b = Batch(7, 4, 2, 64, 16, [50, 48, 60, 51], new=[3, 3, 3, 1], width=3)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_views_scales_and_outputs():
    b = Batch(8, 6, 2, 128, 32, [77, 200, 3], new=[4, 50, 1], q_std=1.0)
    first = b.run()
    b.check(first)
    assert torch.equal(first, b.run(views=False))
    # a slice of a merged projection; rows at odd addresses; heads first
    wide = torch.zeros(b.q.shape[0], 6 * 128 + 64, dtype=b.io, device=DEV)
    for offset in (0, 8, 3):
        view = wide[:, offset:offset + 6 * 128].unflatten(1, (6, 128))
        view.copy_(b.q)
        assert torch.equal(first, b.run(q=view))
    assert torch.equal(first, b.run(q=b.q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)))
    out = torch.full((b.q.shape[0], 8 * 128), 9.0, dtype=b.io, device=DEV)
    b.run(out=out[:, 64:64 + 6 * 128].unflatten(1, (6, 128)))
    assert torch.equal(out[:, 64:64 + 6 * 128].unflatten(1, (6, 128)), first)
    assert (out[:, :64] == 9).all() and (out[:, 64 + 6 * 128:] == 9).all()
    for scale in (0.01, 1.0):
        out, lse = b.run(scale=scale, return_lse=True)
        b.check(out, lse, scale=scale)


def test_large_scores():
    """Weights that are all but zero beside the largest, maxima that rise late and fall."""
    b = Batch(9, 8, 2, 64, 16, [400, 333], q_std=8.0)
    b.k[b.table[0, :25].clamp_min(0)] *= torch.linspace(0.01, 6, 25)[:, None, None, None].to(b.io)
    b.k[b.table[1, :20].clamp_min(0)] *= torch.linspace(6, 0.01, 20)[:, None, None, None].to(b.io)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_not_finite_keys_and_values_reach_whom_they_concern():
    """A NaN key or an infinite value among the positions: the tokens that see it, no other."""
    for heads, kv_heads, dim in ((4, 2, 64), (16, 2, 256)):
        for what in ("k", "v"):
            b = Batch(10, heads, kv_heads, dim, 16, [90, 120, 60], new=[40, 1, 3])
            clean = b.run().cpu()
            at = 70  # of the first request: seen by its last 20 tokens
            getattr(b, what)[b.table[0, at // 16], at % 16, 1, 5] = math.nan if what == "k" else math.inf
            got = b.run().cpu()
            per = heads // kv_heads
            hit = torch.zeros(44, heads, dtype=torch.bool)
            hit[20:40, per:] = True
            assert torch.equal(got[~hit], clean[~hit]), (heads, what)
            assert (~got[hit].isfinite()).any(-1).all()


def test_query_that_is_not_finite():
    b = Batch(11, 8, 2, 128, 16, [100, 50], new=[20, 2])
    clean = b.run().cpu()
    b.q[3, 2, 7] = math.nan
    got = b.run().cpu()
    hit = torch.zeros(22, 8, dtype=torch.bool)
    hit[3, 2] = True
    assert torch.equal(got[~hit], clean[~hit]) and got[3, 2].isnan().all()


def test_rows_do_not_depend_on_their_neighbours():
    """The same request beside others of any length gives the same bits."""
    b = Batch(12, 16, 2, 256, 64, [200, 64, 90], shared=[64])
    alone = b.run().cpu()
    assert torch.equal(alone, b.run().cpu())
    b.q[1:] = 50 * b.q[1:]  # other maxima in the same tiles
    assert torch.equal(b.run().cpu()[0], alone[0])


def test_more_segments_than_threads():
    """700 requests in 30 groups, some of them empty."""
    n = 700
    bounds = [0] + sorted(torch.randint(0, n + 1, (29,), generator=gen(13)).tolist()) + [n]
    lens = [32 + (r * 13) % 50 for r in range(n)]
    b = Batch(13, 2, 1, 64, 16, lens, shared=[32] * 30, groups=bounds)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_far_pages_of_a_large_cache():
    """Pages whose byte offsets pass 32 bits."""
    from logssms_amd.kernel import paged_attention
    pages, page, heads, dim = 5000, 256, 8, 256
    storage = torch.empty(pages, 2, page, heads, dim, dtype=torch.bfloat16, device=DEV)  # 10 GB
    table = torch.tensor([[4999, 3], [2500, 4998]])
    small = Batch(14, 8, 8, 256, 256, [300, 512])
    for a, b in zip(table.flatten().tolist(), small.table.flatten().tolist()):
        storage[a, 0], storage[a, 1] = small.k[b].to(DEV), small.v[b].to(DEV)
    got = paged_attention(small.q.to(DEV), storage[:, 0], storage[:, 1], table.to(DEV), torch.tensor([300, 512]).to(DEV))
    small.check(got)


def test_nothing_to_do():
    from logssms_amd.kernel import paged_attention
    cache = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    q = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    out, lse = paged_attention(q, cache, cache, none.view(0, 1), none, return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    # an empty cache, and a table without room
    q = torch.ones(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    lens = torch.tensor([3, 0], dtype=torch.int32, device=DEV)
    out = paged_attention(q, cache[:0], cache[:0], torch.zeros(2, 1, dtype=torch.int32, device=DEV), lens)
    assert (out == 0).all()
    out, lse = paged_attention(q, cache, cache, torch.zeros(2, 0, dtype=torch.int32, device=DEV), lens, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_graphs_follow_lengths_and_pages():
    """Two graphs and eager calls by turns, lengths and tables changed between replays."""
    from logssms_amd.kernel import paged_attention
    batches = [Batch(20, 16, 2, 256, 64, [64 * 4] * 6, shared=[128]), Batch(21, 8, 2, 128, 16, [80] * 3, new=[8, 40, 1])]
    graphs = []
    for b in batches:
        b.k, b.v = b.k.nan_to_num(0.5), b.v.nan_to_num(0.5, 0.5, 0.5)
        b.on = dict(q=b.q.to(DEV), caches=b.caches(), table=b.table.to(DEV), lens=torch.tensor(b.lens, device=DEV),
                    kw={n: None if t is None else t.to(DEV) for n, t in
                        (("shared_lens", b.shared), ("group_offsets", b.groups), ("cu_seqlens", b.cu))})
        call = lambda b=b: paged_attention(b.on["q"], *b.on["caches"], b.on["table"], b.on["lens"], **b.on["kw"])  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out, call, b))
    for i in range(4):
        for graph, out, call, b in graphs:
            b.on["lens"].sub_(9)
            b.on["table"].copy_(b.on["table"].roll(i, 0))
            if b.shared is not None:
                b.on["table"][:, :2] = b.on["table"][:1, :2]
            graph.replay()
        for graph, out, call, b in graphs:
            got = out.clone()
            assert torch.equal(got, call())
            torch.cuda.synchronize()


def test_another_stream():
    b = Batch(22, 8, 2, 128, 16, [500, 100, 30], new=[3, 60, 1])
    want = b.run()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [b.run() for _ in range(3)]
    stream.synchronize()
    assert all(torch.equal(want, x) for x in got)


def test_pool_appends_and_attention_together():
    """Prompts and then single tokens through a hybrid block pool that holds recurrent states as well:
    keys appended with their rotation, the shared prompt written once, the states untouched."""
    from types import SimpleNamespace

    from logssms_amd.cache import HybridBlockLayout, HybridBlockPool
    from logssms_amd.kernel import append_paged_kv, paged_attention, rotary_embedding
    g = gen(30)
    heads, kv_heads, dim, page, lane = 8, 2, 128, 64, 1
    spec = SimpleNamespace(num_layers=2, state_shape=(2, 64, 64), conv_shape=(512, 3))
    layout = HybridBlockLayout.make(2, spec, kv_heads=kv_heads, head_dim=dim, block_size=page)
    pool = HybridBlockPool(layout, 40, DEV, torch.bfloat16)
    state = pool.allocate_state()
    pool.recurrent_state[pool._starts(state)[0]] = 3.0
    held = pool.state_blocks[state]
    k_cache, v_cache = pool.kv_cache(lane)
    rotary = rotary_embedding(32, 1e4, device=DEV)
    prefix, own = 128, [1, 30, 70]
    first = [pool.allocator.take_run(1) for _ in range(prefix // page)]
    rows = [first + [pool.allocator.take_run(1) for _ in range(2)] for _ in own]
    table = torch.tensor(rows)
    keys, values = [torch.zeros(0, kv_heads, dim, dtype=torch.float64) for _ in range(2)]
    history = [(keys, values) for _ in own]

    def step(requests, starts, counts, shared):
        """The requests' next tokens: appended, then attended to."""
        tokens = sum(counts)
        qkv = randn(tokens, heads + 2 * kv_heads, dim, g=g).to(torch.bfloat16)
        on = qkv.to(DEV)
        q, k, v = on.split([heads, kv_heads, kv_heads], dim=1)
        at = [torch.arange(s, s + c) for s, c in zip(starts, counts)]
        slots = torch.cat([table[r, p // page] * page + p % page for r, p in zip(requests, at)])
        positions = torch.cat(at)
        turned = append_paged_kv(k, v, k_cache, v_cache, slots.to(DEV), positions=positions.to(DEV), rotary=rotary, q=q)
        cu = torch.tensor([0] + counts).cumsum(0)
        out = paged_attention(turned, k_cache, v_cache, table[requests].to(DEV),
                              torch.tensor([s + c for s, c in zip(starts, counts)]).to(DEV),
                              shared_lens=torch.tensor([shared]).to(DEV),
                              cu_seqlens=None if counts == [1] * len(counts) else cu.to(DEV))
        # oracle on what the kernels wrote: the rotated rows as they are in the io type
        keys = ref.rotary(qkv[:, heads:heads + kv_heads], positions, rotary.turns.cpu(), False, 1.0)
        written = k_cache.cpu().reshape(-1, kv_heads, dim)[slots]
        assert ((written.double() - keys).abs() <= ref.rotary_bound(qkv[:, heads:heads + kv_heads], rotary.turns.cpu(), False,
                                                                    1.0, torch.bfloat16, keys)).all()
        want, _, bound, _ = ref.attention(turned.cpu(), k_cache.cpu(), v_cache.cpu(), table[requests],
                                          [s + c for s, c in zip(starts, counts)], cu, dim ** -0.5)
        assert ((out.double().cpu() - want).abs() <= ref.attention_bound(want, bound, torch.bfloat16)).all()

    step([0], [0], [prefix], 0)  # the prompt that all share, once
    step([0, 1, 2], [prefix] * 3, own, prefix)
    for i in range(3):
        step([0, 1, 2], [prefix + n + i for n in own], [1, 1, 1], prefix)
    assert (pool.storage[:, list(held)].view(2, len(held), -1) != 0).any()
    assert (pool.recurrent_state[pool._starts(state)[0]] == 3).all()


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 1, 256), (16, 1, 128), (32, 2, 64)])
def test_prompts_of_many_tiles(io, heads, kv_heads, dim):
    """Tiles of rows that are no multiple of eight, their last ones in part, behind keys in several ranges."""
    b = Batch(40 + dim, heads, kv_heads, dim, 64, [75, 2900, 73 + 5], new=[75, 140, 73], io=io)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("dim", [64, 256])
def test_prompts_behind_a_shared_prefix(dim):
    """All of their tokens are rows of the shared part; one of them ends inside it."""
    b = Batch(41, 16, 2, dim, 64, [640 + 50, 640 + 33, 640 + 1, 600], new=[50, 30, 1, 20], shared=[640])
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def requests_over(b, n):
    """n requests over the pages of the only one of `b`, in another order each."""
    b.table = torch.stack([b.table[0].roll(3 * r) for r in range(n)])
    b.lens = [b.lens[0] - 5 * r for r in range(n)]
    b.q = randn(n, *b.q.shape[1:], g=gen(n)).to(b.io)
    return b


@pytest.mark.parametrize("heads,kv_heads,dim,n", [(8, 8, 256, 128), (320, 8, 256, 32), (320, 8, 64, 64)])
def test_long_ranges_of_keys(heads, kv_heads, dim, n):
    """A block's or wave's keys go on past what one lookup in the table serves; the first and the last
    request stand for all."""
    b = requests_over(Batch(42, heads, kv_heads, dim, 16, [4096 + 5 * n]), n)
    out, lse = b.run(return_lse=True)
    q, table, lens = b.q, b.table, b.lens
    for r in (0, n - 1):
        b.q, b.table, b.lens = q[r:r + 1], table[r:r + 1], lens[r:r + 1]
        b.check(out[r:r + 1], lse[r:r + 1])


def test_more_segments_of_many_rows_than_threads():
    lens = [48 + (r * 29) % 90 for r in range(300)]
    b = Batch(43, 36, 1, 64, 16, lens, shared=[48, 48, 0], groups=[0, 120, 121, 290])
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("heads", [2, 16])
def test_many_empty_requests_in_a_group(heads):
    """Few and many rows of a shared part, the tokens' requests far apart."""
    new = [0] * 150
    new[0], new[1], new[90], new[149] = 2, 1, 3, 1
    lens = [64 + (7 * r) % 40 for r in range(150)]
    b = Batch(44, heads, 1, 128, 16, lens, new=new, shared=[64])
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_thousands_of_requests():
    new = [int(r % 3 != 1) for r in range(5000)]
    lens = [16 + r % 23 for r in range(5000)]
    b = Batch(45, 1, 1, 64, 16, lens, new=new, shared=[16, 16], groups=[7, 4500, 4990])
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_two_streams_at_once():
    """Each call has a workspace of its own."""
    batches = [Batch(46, 16, 2, 256, 64, [900, 4000, 30], new=[3, 200, 1]), Batch(47, 8, 8, 128, 16, [700] * 40)]
    want = [b.run() for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for _ in range(5):
        for b, stream, results in zip(batches, streams, got):
            with torch.cuda.stream(stream):
                results.append(b.run())
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        assert all(torch.equal(w, x) for x in results)


def test_tables_and_lengths_that_are_views():
    from logssms_amd.kernel import paged_attention
    b = Batch(48, 8, 2, 128, 16, [100, 333, 7])
    want = b.run()
    wide = torch.full((6, b.width + 5), 10 ** 6, device=DEV)
    wide[::2, 2:2 + b.width] = b.table.to(DEV)
    lens = torch.tensor(b.lens, device=DEV)
    got = paged_attention(b.q.to(DEV), *b.caches(), wide[::2, 2:2 + b.width], lens)
    assert torch.equal(got, want)


def test_indices_past_32_bits():
    """Pages and lengths whose low halves would be others."""
    b = Batch(49, 8, 2, 128, 16, [100, 64, 200, 33], new=[2, 40, 1, 3], shared=[32])
    b.k, b.v = b.k.nan_to_num(0.5), b.v.nan_to_num(0.5, 0.5, 0.5)
    b.table[:, 1] += 2 ** 32
    b.table[2, 9] -= 2 ** 40
    b.lens[0], b.lens[3] = 2 ** 32 + 5, -(2 ** 33) + 9
    out, lse = b.run(index=torch.int64, return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("heads", [3, 40])
def test_empty_requests_and_tokens_of_nobody(heads):
    """Few and many heads to a key head, requests without tokens among the others, at the start and the end."""
    b = Batch(50, heads, 1, 64, 16, [20, 30, 9, 70, 64, 5], new=[0, 2, 0, 1, 3, 0], shared=[16, 64], groups=[1, 3, 5])
    b.table[2, 0] = b.table[1, 0]
    b.cu = b.cu + 2
    b.q = torch.cat([b.q[:2], b.q, b.q[:1]])
    for _ in range(3):
        out = torch.full(b.q.shape, 7.0, dtype=b.io, device=DEV)
        b.run(out=out)
        out = out.cpu()
        assert (out[:2] == 7).all() and (out[8:] == 7).all()
        want, _, bound, _ = ref.attention(b.q, b.k, b.v, b.table, b.lens, b.cu, 0.125)
        assert ((out.double() - want).abs() <= ref.attention_bound(want, bound, b.io))[2:8].all()


@pytest.mark.parametrize("requests", [1, 62, 63, 64, 65, 255, 256])
@pytest.mark.parametrize("new", [1, 4])
def test_as_many_segments_as_lanes_and_threads(requests, new):
    """One more or fewer than are counted at once; a group, and tokens of nobody's group."""
    lens = [32 + (5 * r) % 40 + new for r in range(requests)]
    b = Batch(51 + requests, 4, 2, 64, 16, lens, new=None if new == 1 else [new] * requests, shared=[32],
              groups=[requests // 3, requests])
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("heads,kv_heads,dim,io", [(48, 16, 64, "f16"), (48, 16, 128, "bf16"), (16, 4, 256, "bf16")])
def test_ragged_prompts_in_several_rounds(heads, kv_heads, dim, io):
    """More tiles than run at once, of all lengths."""
    new = [300, 40, 200, 1, 150, 60]
    lens = [512 + n + 17 * i for i, n in enumerate(new)]
    b = Batch(60 + dim, heads, kv_heads, dim, 64, lens, new=new, shared=[512], io=io)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_many_segments_in_several_rounds():
    """More of many rows than threads, several to a block."""
    lens = [20 + (r * 37) % 60 for r in range(300)]
    b = Batch(61, 66, 2, 256, 16, lens)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (16, 2, 256), (80, 2, 128)])
@pytest.mark.parametrize("lens,new,shared", [
    ([90, 16, 40, 9], None, None), ([5000, 3000, 4001], None, None), ([90, 3, 70, 40], [40, 5, 70, 1], None),
    ([160 + 20, 160 + 7, 160 + 30], [20, 3, 1], [160])])
def test_scores_of_minus_infinity(io, heads, kv_heads, dim, lens, new, shared):
    """A token all of whose scores are so gives NaN, as their softmax is, also where it is put together
    from pieces; weights of some of them are zero; a token that sees nothing gives zeros all the same."""
    b = Batch(53, heads, kv_heads, dim, 16, lens, new=new, shared=shared, io=io)
    b.q[..., 5] = b.q[..., 5].abs() + 1
    cu = b.cu if b.cu is not None else torch.arange(len(lens) + 1)
    clean, k = b.run().cpu(), b.k.clone()
    per = heads // kv_heads
    # all of request 1's
    own = torch.zeros(b.q.shape[0], heads, dtype=torch.bool)
    own[cu[1]:cu[2], per:] = True
    for p in range(lens[1]):
        b.k[b.table[1, p // 16], p % 16, 1, 5] = -math.inf
    hit = own.clone()
    if shared is None:
        for t in range(int(cu[1]), int(cu[2])):  # those before its first position
            hit[t] &= lens[1] - (int(cu[2]) - 1 - t) > 0
    out, lse = b.run(return_lse=True)
    out, lse = out.cpu(), lse.cpu()
    assert out[hit].isnan().all() and (lse[hit] == -math.inf).all()
    assert (out[own & ~hit] == 0).all()
    if shared is None:
        assert torch.equal(out[~own], clean[~own])
        # every other one of request 2's, the first among them: as good as scores that are far below the others
        results = []
        for value in (-math.inf, -3.0e4):
            b.k = k.clone()
            for p in range(0, lens[2], 2):
                b.k[b.table[2, p // 16], p % 16, 1, 5] = value
            results.append(b.run(return_lse=True))
        seen = torch.ones(b.q.shape[0], heads, dtype=torch.bool)  # more than the first position
        for t in range(int(cu[2]), int(cu[3])):
            if lens[2] - (int(cu[3]) - 1 - t) == 1:
                seen[t, per:] = False
                assert results[0][0].cpu()[t, per:].isnan().all()
        assert torch.equal(results[0][0].cpu()[seen], results[1][0].cpu()[seen])
        assert torch.equal(results[0][1].cpu()[seen], results[1][1].cpu()[seen])
    else:  # whoever shares them sees some others as well, or none
        others = torch.zeros_like(own)
        others[:, per:] = True
        assert torch.equal(out[~others], clean[~others])
        assert out[~own].isfinite().all()


def test_neighbours_of_other_lengths():
    """A row's last bits may follow where the keys are cut, which the lengths beside it decide: it stays
    within its bound."""
    b = Batch(54, 16, 2, 256, 64, [200, 6000, 900, 70], shared=[64])
    for others in ((6000, 900, 70), (64, 64, 64), (6000, 0, 1), (70, 900, 0), (0, 0, 0)):
        b.lens = [200, *others]
        out, lse = b.run(return_lse=True)
        b.check(out, lse)


@pytest.mark.parametrize("heads,kv_heads,dim,lens,new,shared", [
    (8, 2, 128, [500, 33, 70], None, None), (16, 2, 256, [400, 90, 130], [60, 1, 9], [64]),
    (12, 4, 64, [64 + 3, 64 + 40, 64], [3, 40, 1], [64])])
def test_caches_of_other_layouts(heads, kv_heads, dim, lens, new, shared):
    """Heads first, tokens of all pages side by side, room between rows and pages, keys and values each
    in a layout of its own."""
    from logssms_amd.kernel import paged_attention
    page = 32
    b = Batch(55, heads, kv_heads, dim, page, lens, new=new, shared=shared)
    want, want_lse = b.run(return_lse=True)
    b.check(want, want_lse)

    def laid_out(x, order, pad):
        """`x` with its axes in this order in memory, `pad` more elements behind each row."""
        at = x.permute(order)
        room = torch.full((*at.shape[:-1], at.shape[-1] + pad), math.nan, dtype=x.dtype, device=DEV)
        view = room[..., :at.shape[-1]]
        view.copy_(at)
        return view.permute([order.index(d) for d in range(4)])

    layouts = [((0, 2, 1, 3), 0), ((2, 0, 1, 3), 0), ((1, 0, 2, 3), 8), ((0, 1, 2, 3), 24)]
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    for k_layout, v_layout in zip(layouts + [((0, 1, 2, 3), 0)], layouts[::-1] + [((0, 2, 1, 3), 0)]):
        k, v = laid_out(b.k, *k_layout), laid_out(b.v, *v_layout)
        assert torch.equal(k.cpu().nan_to_num(), b.k.nan_to_num())
        out, lse = paged_attention(b.q.to(DEV), k, v, b.table.to(DEV), torch.tensor(lens).to(DEV),
                                   shared_lens=on(b.shared), cu_seqlens=on(b.cu), return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), (k_layout, v_layout)
