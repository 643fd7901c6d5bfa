"""Measured cases of the full-attention layers beside the Gated DeltaNet ones:
rotary positions, appending keys and values to a paged cache with the rotation
on the way, and the attention that reads this cache for a batch whose requests
share a prefix.

The cache is that of ``HybridBlockPool``: a page holds the keys of its tokens,
then their values, ``[tokens, kv heads, head dim]`` each.  Head layouts are those
of the hybrid model that the benchmark's layer belongs to (16 query and 2 key
heads of 256 channels, 64 of them rotated) and generic ones; batches are those
of the benchmark (1, 37 and 256 decoding sequences, 64 x 8 drafted tokens, 16384
prompt tokens).
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _heads(q=16, kv=2, dim=256):
    return {"heads": q, "kv_heads": kv, "dim": dim}


def listed():
    full = _heads()
    return [
        # one user's next token: latency
        {"name": "rotary_1", "op": "rotary", "tokens": 1, **full, "rotated": 64, "interleaved": False, "base": 1e7,
         "scaling": "none", "factor": 1.0, "start": 5000, "io": "bf16"},
        # a ragged prompt, far into a context stretched eightfold, every channel rotated, pairs side by side
        {"name": "rotary_777_far", "op": "rotary", "tokens": 777, **_heads(32, 8, 128), "rotated": 128,
         "interleaved": True, "base": 1e4, "scaling": "yarn", "factor": 8.0, "start": 900000, "io": "f16"},
        # the prefill benchmark's tokens
        {"name": "rotary_16384", "op": "rotary", "tokens": 16384, **full, "rotated": 64, "interleaved": False,
         "base": 1e7, "scaling": "none", "factor": 1.0, "start": 0, "io": "bf16"},
        # the new keys and values of a decode batch, its queries rotated with them
        {"name": "append_256", "op": "append", "tokens": 256, **full, "rotated": 64, "interleaved": False, "base": 1e7,
         "scaling": "none", "factor": 1.0, "start": 30000, "page": 64, "padded": 0, "queries": True, "io": "bf16"},
        # a padded batch without positions: rows of slot -1 are left out
        {"name": "append_1500_f16", "op": "append", "tokens": 1500, **_heads(8, 8, 64), "rotated": 0,
         "interleaved": False, "base": 1e4, "scaling": "none", "factor": 1.0, "start": 0, "page": 16, "padded": 36,
         "queries": False, "io": "f16"},
        # the prompts of the prefill benchmark
        {"name": "append_16384", "op": "append", "tokens": 16384, **full, "rotated": 64, "interleaved": False,
         "base": 1e7, "scaling": "linear", "factor": 4.0, "start": 0, "page": 64, "padded": 0, "queries": True,
         "io": "bf16"},
        # one sequence's next token behind 4096 others: latency
        {"name": "attend_1", "op": "attend", "requests": 1, "groups": 1, "shared": 0, "own_from": 4097, "own_to": 4097,
         "new_from": 1, "new_to": 1, **full, "page": 64, "io": "bf16"},
        # an odd decode batch of short chats, nothing shared, as many key heads as query heads
        {"name": "attend_37_f16", "op": "attend", "requests": 37, "groups": 1, "shared": 0, "own_from": 1, "own_to": 700,
         "new_from": 1, "new_to": 1, **_heads(8, 8, 64), "page": 16, "io": "f16"},
        # 256 sequences that ask about one document
        {"name": "attend_256_shared", "op": "attend", "requests": 256, "groups": 1, "shared": 32768, "own_from": 1, "own_to": 1024,
         "new_from": 1, "new_to": 1, **full, "page": 64, "io": "bf16"},
        # 64 sequences of 8 drafts behind four system prompts
        {"name": "attend_64x8_groups", "op": "attend", "requests": 64, "groups": 4, "shared": 2500, "own_from": 64, "own_to": 4096,
         "new_from": 8, "new_to": 8, **_heads(32, 8, 128), "page": 128, "io": "bf16"},
        # prompts of all lengths behind a shared one, some of them continued
        {"name": "attend_prompts", "op": "attend", "requests": 6, "groups": 1, "shared": 8192, "own_from": 2, "own_to": 4000,
         "new_from": 1, "new_to": 2048, **full, "page": 64, "io": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend"])
    heads = rng.choice([(16, 2, 256), (16, 2, 256), (32, 8, 128), (8, 8, 64), (12, 4, 128), (7, 1, 64), (24, 2, 128)])
    case = {"op": op, **_heads(*heads), "io": rng.choice(["bf16", "bf16", "f16"])}
    if op != "attend":
        tokens = _log_int(rng, 1, min(16384, 16384 * 18 * 256 // ((heads[0] + 2 * heads[1]) * heads[2])))
        rotated = rng.choice([heads[2], heads[2] // 2, heads[2] // 4])
        scaling = rng.choice(["none", "none", "linear", "base", "wavelength", "yarn"])
        case.update(tokens=tokens, rotated=rotated, interleaved=rng.random() < 0.4, base=rng.choice([1e4, 5e5, 1e7]),
                    scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
                    start=_log_int(rng, 1, 1000000))
        if op == "append":
            case.update(page=rng.choice([16, 64, 128, 192, 1088]), padded=rng.choice([0, 0, rng.randint(0, tokens // 4)]),
                        queries=rng.random() < 0.7)
        return case
    groups = rng.choice([1, 1, 1, 2, 4])
    kind = rng.choice(["decode", "decode", "drafts", "prompts"])
    new_from, new_to = {"decode": (1, 1), "drafts": (rng.randint(2, 9),) * 2, "prompts": (1, _log_int(rng, 16, 2048))}[kind]
    own_to = _log_int(rng, max(new_to, 8), 8192)
    case.update(requests=max(groups, _log_int(rng, 1, {"decode": 256, "drafts": 64, "prompts": 6}[kind])), groups=groups,
                own_from=min(own_to, max(new_to, rng.choice([1, own_to // 8]))), own_to=own_to, new_from=new_from,
                new_to=new_to, shared=0 if rng.random() < 0.3 else _log_int(rng, 16, 32768),
                page=rng.choice([16, 64, 64, 128, 192, 1088]))
    largest = work(listed()[-1])["flops"]
    while work(case)["flops"] > largest or _keys_held(case) > 400000:  # no dearer than the largest listed one
        case["requests"] = max(groups, case["requests"] // 2)
        case["shared"] //= 2
        case["own_from"], case["own_to"] = max(new_to, case["own_from"] // 2), max(new_to, case["own_to"] // 2)
    return case


# ------------------------------------------------------------------ sizes of a batch

def _lengths(case):
    """New tokens, own positions (the new ones among them) of every request, the
    first request and the shared positions of every group, in whole pages: of the
    case, the same for every seed."""
    rng = random.Random(17 * case["requests"] + case["own_to"])
    new = [_log_int(rng, case["new_from"], case["new_to"]) for _ in range(case["requests"])]
    lengths = [max(n, _log_int(rng, case["own_from"], case["own_to"])) for n in new]
    if case["new_from"] != case["new_to"]:  # prompts: some start right behind the shared one
        lengths = [n if i % 2 else length for i, (n, length) in enumerate(zip(new, lengths))]
    r, g = case["requests"], case["groups"]
    first = [r * i // g for i in range(g + 1)]
    shared = [max(0, case["shared"] - 100 * i) // case["page"] * case["page"] for i in range(g)]
    return new, lengths, first, shared


def _keys_held(case):
    _, lengths, _, shared = _lengths(case)
    return (sum(lengths) + sum(shared)) * case["kv_heads"] * case["dim"] // 512


# ------------------------------------------------------------------ inputs

def _randn(g, *shape, std=1.0):
    return torch.empty(*shape, device=DEV).normal_(0.0, std, generator=g)


def _turns(case):
    """Revolutions per position of each rotated pair, in 64 bits, and the factor
    on the rotated values: the plain frequencies and four ways to stretch them
    (every position, the base, by wavelength, by a ramp over the pairs)."""
    n, base, factor = case["rotated"], case["base"], case["factor"]
    i = torch.arange(0, n, 2, dtype=torch.float64)
    if case["scaling"] == "base":
        base = base * factor ** (n / max(n - 2, 1))
    turns = base ** (-i / n) / (2 * math.pi)
    scale = 1.0
    if case["scaling"] == "linear":
        turns = turns / factor
    elif case["scaling"] == "wavelength":
        kept = ((8192 * turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        turns = turns * kept + turns / factor * (1 - kept)
    elif case["scaling"] == "yarn":
        def pair(rotations):  # the pair that turns so often over the original length
            return n * math.log(8192 / (rotations * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), n - 1)
        kept = 1 - ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        turns = turns * kept + turns / factor * (1 - kept)
        scale = 0.1 * math.log(factor) + 1.0
    return turns.to(DEV), scale


def _cache(g, pages, page, kv_heads, dim, io):
    storage = _randn(g, pages, 2, page, kv_heads, dim).to(io)
    return storage[:, 0], storage[:, 1]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    io = DTYPES[case["io"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case}
    if case["op"] in ("rotary", "append"):
        tokens = case["tokens"]
        # column slices of the merged projection
        merged = _randn(g, tokens, (heads + 2 * kv_heads) * dim).to(io).view(tokens, heads + 2 * kv_heads, dim)
        state["q"], state["k"], state["v"] = merged.split([heads, kv_heads, kv_heads], dim=1)
        jump = torch.randint(0, 3, (tokens,), device=DEV, generator=g).cumsum(0) if case["op"] == "append" else \
            torch.arange(tokens, device=DEV)
        state["positions"] = (case["start"] + jump).to(torch.int32)
        if case["rotated"]:
            if own:
                from logssms_amd.kernel import rotary_embedding
                state["rotary"] = rotary_embedding(case["rotated"], case["base"], interleaved=case["interleaved"],
                                                   scaling=case["scaling"], factor=case["factor"],
                                                   original_length=8192, device=DEV)
            state["turns"], state["scale"] = _turns(case)
    if case["op"] == "append":
        page = case["page"]
        pages = -(-tokens // page) + 5
        state["k_cache"], state["v_cache"] = _cache(g, pages, page, kv_heads, dim, io)
        # whole pages in any order, token after token inside them
        order = torch.randperm(pages, device=DEV, generator=g)
        at = torch.arange(tokens, device=DEV)
        slots = order[at // page] * page + at % page
        slots[tokens - case["padded"]:] = -1
        state["slots"] = slots
    if case["op"] == "attend":
        new, lengths, first, shared = _lengths(case)
        page = case["page"]
        own_pages = [-(-n // page) for n in lengths]
        total = sum(own_pages) + sum(n // page for n in shared)
        order = torch.randperm(total + 3, device=DEV, generator=g).cpu().tolist()
        rows, seq_lens = [], []
        for j, n in enumerate(shared):
            prefix = [order.pop() for _ in range(n // page)]
            for r in range(first[j], first[j + 1]):
                rows.append(prefix + [order.pop() for _ in range(own_pages[r])])
                seq_lens.append(n + lengths[r])
        width = max(len(row) for row in rows)
        state["page_table"] = torch.tensor([row + [-1] * (width - len(row)) for row in rows], dtype=torch.int32).to(DEV)
        state["seq_lens"] = torch.tensor(seq_lens, dtype=torch.int32).to(DEV)
        state["shared_lens"] = torch.tensor(shared, dtype=torch.int32).to(DEV)
        state["group_offsets"] = torch.tensor(first, dtype=torch.int32).to(DEV)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state["cu_seqlens"] = None if case["new_to"] == 1 else torch.tensor(starts, dtype=torch.int32).to(DEV)
        # queries and keys as they come out of their norms: a few keys stand out for each query
        state["q"] = _randn(g, starts[-1], heads, dim, std=2.0).to(io)
        state["k_cache"], state["v_cache"] = _cache(g, total + 3, page, kv_heads, dim, io)
        # what the host knows of the batch
        state["sizes"] = (starts, seq_lens, shared, first)
    return state


# ------------------------------------------------------------------ one pass

def _run_own(state):
    from logssms_amd import kernel
    case = state["case"]
    if case["op"] == "rotary":
        return kernel.apply_rotary(state["q"], state["k"], state["positions"], state["rotary"])
    if case["op"] == "append":
        rotary = state.get("rotary")
        q = kernel.append_paged_kv(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slots"],
                                   positions=None if rotary is None else state["positions"], rotary=rotary,
                                   q=state["q"] if case["queries"] else None)
        return [state["k_cache"], state["v_cache"]] + ([q] if case["queries"] else [])
    return kernel.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"],
                                  state["seq_lens"], shared_lens=state["shared_lens"],
                                  group_offsets=state["group_offsets"], cu_seqlens=state["cu_seqlens"])


def _rotate(x, positions, turns, scale, interleaved):
    """fp32 result; angles in 64 bits."""
    n = 2 * turns.numel()
    angle = positions.double()[:, None, None] * turns * (2 * math.pi)
    cos, sin = torch.cos(angle).float() * scale, torch.sin(angle).float() * scale
    x = x.float()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2] = a * cos - b * sin
        y[..., 1:n:2] = b * cos + a * sin
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2] = a * cos - b * sin
        y[..., n // 2:n] = b * cos + a * sin
    return y


def _plain_attend(state):
    """Group by group: scores of the shared keys for all rows at once, scores of
    each request's own keys, one softmax over both, the two products' sum."""
    case = state["case"]
    starts, seq_lens, shared, first = state["sizes"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    per = heads // kv_heads
    out = torch.empty_like(state["q"])
    k_cache, v_cache, table = state["k_cache"], state["v_cache"], state["page_table"].long()
    for j, prefix in enumerate(shared):
        r0, r1 = first[j], first[j + 1]
        if r0 == r1:
            continue
        n = r1 - r0
        count = [starts[r + 1] - starts[r] for r in range(r0, r1)]
        most, longest = max(count), max(seq_lens[r0:r1]) - prefix
        step = torch.arange(most, device=DEV)
        begin = torch.tensor(starts[r0:r1], device=DEV)[:, None]
        length = torch.tensor(seq_lens[r0:r1], device=DEV)[:, None]
        queries = torch.tensor(count, device=DEV)[:, None]
        token = begin + torch.minimum(step, queries - 1)  # [n, most], the last one again where there are fewer
        q = state["q"][token].float().view(n, most, kv_heads, per, dim) * dim ** -0.5
        at = prefix + torch.arange(longest, device=DEV)
        pages = table[r0:r1, (at // page).clamp_max(table.shape[1] - 1)].clamp_min(0)  # [n, longest]
        ko, vo = k_cache[pages, at % page].float(), v_cache[pages, at % page].float()
        so = q.permute(0, 2, 1, 3, 4).reshape(n, kv_heads, most * per, dim) @ ko.permute(0, 2, 3, 1)
        seen = at[None, None, :] <= (length - queries + step)[:, :, None]  # [n, most, longest]
        so = torch.where(seen.repeat_interleave(per, 1)[:, None], so, -math.inf)
        top = so.amax(-1, keepdim=True)
        if prefix:
            at = torch.arange(prefix, device=DEV)
            pages = table[r0, at // page]
            kp, vp = k_cache[pages, at % page].float(), v_cache[pages, at % page].float()  # [prefix, kv_heads, dim]
            rows = q.permute(2, 0, 1, 3, 4).reshape(kv_heads, -1, dim)
            sp = (rows @ kp.permute(1, 2, 0)).view(kv_heads, n, most * per, prefix).transpose(0, 1)
            top = torch.maximum(top, sp.amax(-1, keepdim=True))
        eo = torch.exp(so - top)
        y, total = eo @ vo.transpose(1, 2), eo.sum(-1, keepdim=True)
        del so, eo
        if prefix:
            ep = torch.exp(sp - top)
            del sp
            total = total + ep.sum(-1, keepdim=True)
            y = y + (ep.transpose(0, 1).reshape(kv_heads, -1, prefix) @ vp.transpose(0, 1)).view(
                kv_heads, n, most * per, dim).transpose(0, 1)
        y = (y / total).view(n, kv_heads, most, per, dim).transpose(1, 2).reshape(n, most, heads, dim)
        if most == 1:
            out[starts[r0]:starts[r1]] = y[:, 0].to(out.dtype)
        else:
            for i, c in enumerate(count):
                out[starts[r0 + i]:starts[r0 + i] + c] = y[i, :c].to(out.dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    io = DTYPES[case["io"]]
    if case["op"] == "attend":
        return _plain_attend(state)
    rotate = (lambda x: _rotate(x, state["positions"], state["turns"], state["scale"], case["interleaved"]).to(io)) \
        if case["rotated"] else (lambda x: x)
    if case["op"] == "rotary":
        return rotate(state["q"]), rotate(state["k"])
    k, v, slots = rotate(state["k"]), state["v"], state["slots"]
    if case["padded"]:
        wanted = slots >= 0
        k, v, slots = k[wanted], v[wanted], slots[wanted]
    page = case["page"]
    state["k_cache"][slots // page, slots % page] = k
    state["v_cache"][slots // page, slots % page] = v
    return [state["k_cache"], state["v_cache"]] + ([rotate(state["q"])] if case["queries"] else [])


def work(case):
    """Inputs read once, outputs written once; a key and its value once however
    many queries see them."""
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["io"] == "f32" else 2
    if case["op"] == "attend":
        new, lengths, first, shared = _lengths(case)
        keys = sum(lengths) + sum(shared[j] for j in range(len(shared)) if first[j] < first[j + 1])
        seen = 0
        for j, n in enumerate(shared):
            for r in range(first[j], first[j + 1]):
                c = new[r]  # the last of c queries sees all, each before it one less
                seen += c * (n + lengths[r]) - c * (c - 1) // 2
        return {"bytes": size * dim * (2 * sum(new) * heads + 2 * keys * kv_heads) + 4 * len(new),
                "flops": 4 * dim * heads * seen}
    t = case["tokens"]
    if case["op"] == "rotary":
        return {"bytes": t * (2 * size * (heads + kv_heads) * dim + 4), "flops": 3 * t * (heads + kv_heads) * case["rotated"]}
    kept = t - case["padded"]
    queries = heads * t if case["queries"] else 0
    return {"bytes": 2 * size * dim * (queries + 2 * kept * kv_heads) + 12 * t,
            "flops": 3 * case["rotated"] * (queries + kept * kv_heads)}


# ------------------------------------------------------------------ 64 bits

def _rotate64(x, positions, turns, scale, interleaved):
    n = 2 * turns.numel()
    part, rest = x[..., :n].to(torch.float64), x[..., n:].to(torch.float64)
    phase = torch.remainder(positions.to(torch.float64)[:, None] * turns[None, :], 1.0) * (2 * math.pi)
    unit = torch.polar(torch.full_like(phase, scale), phase)[:, None, :]
    if interleaved:
        pairs = torch.view_as_complex(part.reshape(*part.shape[:-1], n // 2, 2).contiguous())
        return torch.cat([torch.view_as_real(pairs * unit).flatten(-2), rest], -1)
    z = torch.complex(part[..., :n // 2], part[..., n // 2:]) * unit
    return torch.cat([z.real, z.imag, rest], -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] != "attend":
        turn = (lambda x: _rotate64(x, state["positions"], state["turns"], state["scale"], case["interleaved"])) \
            if case["rotated"] else (lambda x: x.to(torch.float64))
        if case["op"] == "rotary":
            return turn(state["q"]), turn(state["k"])
        page = case["page"]
        k_cache, v_cache = state["k_cache"].to(torch.float64), state["v_cache"].to(torch.float64)
        flat_k = k_cache.reshape(-1, *k_cache.shape[2:])
        flat_v = v_cache.reshape(-1, *v_cache.shape[2:])
        kept = case["tokens"] - case["padded"]
        flat_k[state["slots"][:kept]] = turn(state["k"])[:kept]
        flat_v[state["slots"][:kept]] = state["v"][:kept].to(torch.float64)
        out = [flat_k.view(-1, page, *flat_k.shape[1:]), flat_v.view(-1, page, *flat_v.shape[1:])]
        return out + ([turn(state["q"])] if case["queries"] else [])
    starts, seq_lens, _, _ = state["sizes"]
    page, per = case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEV)
    for r, length in enumerate(seq_lens):  # each request by itself, over all of its positions
        at = torch.arange(length, device=DEV)
        pages = state["page_table"][r].long()[at // page]
        q = state["q"][starts[r]:starts[r + 1]].to(torch.float64)
        count = q.shape[0]
        for h in range(case["kv_heads"]):
            k = state["k_cache"][pages, at % page, h].to(torch.float64)
            v = state["v_cache"][pages, at % page, h].to(torch.float64)
            for t0 in range(0, count, 512):
                some = q[t0:t0 + 512, h * per:(h + 1) * per]
                s = some.reshape(-1, case["dim"]) @ k.t().contiguous() / math.sqrt(case["dim"])
                hidden = at[None, :] > (length - count + t0 + torch.arange(some.shape[0], device=DEV))[:, None]
                s = s.masked_fill(hidden.repeat_interleave(per, 0), -math.inf)
                y = torch.softmax(s, dim=-1) @ v
                out[starts[r] + t0:starts[r] + t0 + some.shape[0], h * per:(h + 1) * per] = y.view(-1, per, case["dim"])
    return out
