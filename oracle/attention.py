"""Rotary positions, cache appends and paged attention in 64 bits, from their
definitions, with bounds for kernels that compute them in fp32 and round to an io
type.  Plain loops; CPU tensors."""

import math

import torch

F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotary(x, positions, turns, interleaved, scale):
    """[tokens, heads, dim] -> the same in float64."""
    n = 2 * turns.numel()
    angle = torch.remainder(positions.double()[:, None] * turns.double(), 1.0) * (2 * math.pi)
    cos, sin = scale * torch.cos(angle)[:, None], scale * torch.sin(angle)[:, None]
    y = x.double().clone()
    first = slice(0, n, 2) if interleaved else slice(0, n // 2)
    second = slice(1, n, 2) if interleaved else slice(n // 2, n)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first] = a * cos - b * sin
    y[..., second] = a * sin + b * cos
    return y


def rotary_bound(x, turns, interleaved, scale, dtype, want):
    """Of a result in `dtype`: its own rounding, and that of fp32 cosines and sines
    (the angle's fraction rounded once, at most 2 pi / 4 2^-24 ... 2^-22 with the
    functions' own steps), times the scale, two products and their sum."""
    n = 2 * turns.numel()
    first = slice(0, n, 2) if interleaved else slice(0, n // 2)
    second = slice(1, n, 2) if interleaved else slice(n // 2, n)
    size = torch.zeros_like(want)
    both = abs(scale) * (x.double()[..., first].abs() + x.double()[..., second].abs())
    size[..., first], size[..., second] = both, both
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return want.abs() * half_step(dtype) + 1.01 * size * 2.0 ** -21 + tiny


def keys_of(cache, pages, length):
    """Positions 0 .. length - 1 behind a row of the table: [length, kv heads, dim]
    float64, zeros where the page lies outside of the cache."""
    page = cache.shape[1]
    out = torch.zeros(length, *cache.shape[2:], dtype=torch.float64)
    for p in range(0, length, page):
        at = int(pages[p // page])
        n = min(page, length - p)
        if 0 <= at < cache.shape[0]:
            out[p:p + n] = cache[at, :n].double()
    return out


def attention(q, k_cache, v_cache, table, seq_lens, cu, scale):
    """(out, lse, bound): out and lse in float64, rows that no request owns as NaN;
    `bound` on a kernel's error in out, without the rounding of the result."""
    tokens, heads, dim = q.shape
    per = heads // k_cache.shape[2]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    lse = torch.full((tokens, heads), math.nan, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    lse_bound = torch.zeros(tokens, heads, dtype=torch.float64)
    capacity = table.shape[1] * k_cache.shape[1]
    for r in range(table.shape[0]):
        first, last = (int(cu[r]), int(cu[r + 1])) if cu is not None else (r, r + 1)
        length = max(0, min(int(seq_lens[r]), capacity))
        k, v = keys_of(k_cache, table[r], length), keys_of(v_cache, table[r], length)
        for t in range(first, last):
            seen = max(0, min(length, int(seq_lens[r]) - (last - 1 - t)))
            for h in range(heads):
                if seen == 0:
                    out[t, h], lse[t, h] = 0.0, -math.inf
                    continue
                x, keys, values = q[t, h].double(), k[:seen, h // per], v[:seen, h // per]
                s = keys @ x * scale
                p = torch.softmax(s, 0)
                out[t, h], lse[t, h] = p @ values, torch.logsumexp(s, 0)
                # scores: fp32 sums of dim products, then a scaled difference
                off = (dim + 8) * F32 * scale * float((keys.abs() @ x.abs()).max()) + 2.0 ** -20
                size = p @ values.abs()
                # weights off by `off` above and below the line and rounded to the io type, fp32 sums of them
                bound[t, h] = size * (2 * off + half_step(q.dtype) + (seen / 16 + 64) * F32)
                if q.dtype == torch.float16:  # weights below the normal range
                    bound[t, h] += seen * 2.0 ** -25 * values.abs().max()
                lse_bound[t, h] = off + (seen / 16 + 64) * F32 + abs(float(lse[t, h])) * 2.0 ** -22
    return out, lse, bound, lse_bound


def attention_bound(want, bound, dtype):
    """With the rounding of the result."""
    return bound + (want.abs() + bound) * half_step(dtype) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


__all__ = ["attention", "attention_bound", "half_step", "keys_of", "rotary", "rotary_bound"]
