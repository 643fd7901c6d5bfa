"""Measured cases of the 8-bit projection path around a Gated DeltaNet layer:
the residual addition and root-mean-square norm in front of it, the gated norm
behind it, the quantisation of rows, and the block-scaled matrix product that
reads what they write.

Values are ``float8_e4m3fn`` with one fp32 scale for each 128 values of a row
(activations) or each block of 128 x 128 (weights): the represented number is
``value * scale`` and ``scale = max|block| / 448``.

Sizes are those of the benchmark's layer (hidden size 2048, 32 value heads of
128 channels, 12288 columns of the merged q/k/v/z projection, 4096 rows of the
output projection's input; 1, 37 and 256 decoding sequences, 64 x 8 drafted
tokens, 16384 prompt tokens) and odd ones.
"""

import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
TOP = 448.0  # the largest float8_e4m3fn
TINY = 2.0 ** -126  # the least scale, that of a block of zeros
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the norm before a layer while one sequence decodes: latency
        {"name": "add_norm_1", "op": "norm", "tokens": 1, "width": 2048, "io": "bf16", "add": True, "fp8": True, "keep": True},
        # a ragged prompt through a narrow layer without quantised weights
        {"name": "norm_777_f16", "op": "norm", "tokens": 777, "width": 1000, "io": "f16", "add": False, "fp8": False, "keep": True},
        # the norm before a layer over the prefill benchmark's 16384 tokens
        {"name": "add_norm_16384", "op": "norm", "tokens": 16384, "width": 2048, "io": "bf16", "add": True, "fp8": True, "keep": False},
        # the core output of 256 decoding sequences on its way to the output projection
        {"name": "gated_256", "op": "gated", "tokens": 256, "heads": 32, "dim": 128, "io": "bf16"},
        # the core output of the prefill benchmark
        {"name": "gated_16384", "op": "gated", "tokens": 16384, "heads": 32, "dim": 128, "io": "bf16"},
        # rows that no norm has quantised: a small decode batch in f16
        {"name": "quantize_37_f16", "op": "quantize", "tokens": 37, "width": 4096, "io": "f16"},
        # the same over a whole prompt batch
        {"name": "quantize_16384", "op": "quantize", "tokens": 16384, "width": 2048, "io": "bf16"},
        # merged q/k/v/z projection for one decoding sequence: 25 MB of weights for one row
        {"name": "linear_1_in", "op": "linear", "tokens": 1, "n": 12288, "k": 2048, "out": "bf16"},
        # output projection of a small decode batch
        {"name": "linear_37_out", "op": "linear", "tokens": 37, "n": 2048, "k": 4096, "out": "f16"},
        # merged projection of 64 sequences with 8 drafted tokens each
        {"name": "linear_512_in", "op": "linear", "tokens": 512, "n": 12288, "k": 2048, "out": "bf16"},
        # a ragged prompt and sizes that no tile or block divides
        {"name": "linear_2900_odd", "op": "linear", "tokens": 2900, "n": 1111, "k": 1000, "out": "bf16"},
        # merged projection of the prefill benchmark
        {"name": "linear_16384_in", "op": "linear", "tokens": 16384, "n": 12288, "k": 2048, "out": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "gated", "quantize", "linear", "linear", "linear", "linear"])
    io = rng.choice(["bf16", "bf16", "f16"])
    if op in ("norm", "quantize"):
        width = rng.choice([_log_int(rng, 64, 8192), 64 * rng.randint(2, 64), 2048])
        tokens = _log_int(rng, 1, 16384 * 2048 // max(2048, width))
        if op == "quantize":
            return {"op": op, "tokens": tokens, "width": width, "io": io}
        fp8 = rng.random() < 0.7
        return {"op": op, "tokens": tokens, "width": width, "io": io, "add": rng.random() < 0.7, "fp8": fp8,
                "keep": not fp8 or rng.random() < 0.5}
    if op == "gated":
        heads, dim = rng.choice([(32, 128), (32, 128), (16, 128), (8, 64), (5, 96), (4, 32)])
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "heads": heads, "dim": dim, "io": io}
    n, k = rng.choice([(12288, 2048), (2048, 4096), (6144, 1024), (1024, 2048),
                       (_log_int(rng, 16, 12288), _log_int(rng, 32, 8192)),
                       (_log_int(rng, 16, 12288), _log_int(rng, 32, 8192))])
    top = min(16384, 16384 * 12288 * 2048 // (n * k))
    return {"op": op, "tokens": _log_int(rng, 1, top), "n": n, "k": k, "out": io}


# ------------------------------------------------------------------ inputs

def _randn(g, *shape, std=1.0):
    return torch.empty(*shape, device=DEV).normal_(0.0, std, generator=g)


def _hidden(g, tokens, width, std=1.0):
    """Hidden states: normal, with a few channels that are much larger and
    tokens of different sizes, as the activations of trained models have."""
    x = _randn(g, tokens, width, std=std)
    channels = torch.rand(width, device=DEV, generator=g)
    x *= torch.where(channels < 0.01, 12.0, 1.0)
    return x * torch.exp(0.5 * _randn(g, tokens, 1))


def _padded_rows(values):
    """Rows at a stride that is a multiple of 16 bytes, as the quantisers lay them out."""
    rows, width = values.shape
    if width % 16 == 0:
        return values.contiguous()
    wide = torch.zeros(rows, -(-width // 16) * 16, dtype=torch.uint8, device=values.device)
    wide[:, :width] = values.view(torch.uint8)
    return wide.view(torch.float8_e4m3fn)[:, :width]


def _quantize_rows(x):
    """fp32 rows -> float8 values and the scales of their blocks of 128."""
    rows, width = x.shape
    blocks = -(-width // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - width)).view(rows, blocks, BLOCK)
    scales = (x.abs().amax(-1) / TOP).clamp_min(TINY)
    values = (x / scales[:, :, None]).to(torch.float8_e4m3fn).view(rows, blocks * BLOCK)[:, :width]
    return values, scales


def _weight(g, n, k):
    """A projection's weights in float8 with a scale for each block of 128 x 128."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, device=DEV)
    w[:n, :k] = _randn(g, n, k, std=0.02) * torch.exp(0.4 * _randn(g, n, 1))
    w = w.view(nb, BLOCK, kb, BLOCK)
    scales = (w.abs().amax((1, 3)) / TOP).clamp_min(TINY)
    values = (w / scales[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)[:n, :k]
    return _padded_rows(values), scales


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = {"case": case}
    op, tokens = case["op"], case["tokens"]
    if op == "norm":
        io = DTYPES[case["io"]]
        state["x"] = _hidden(g, tokens, case["width"]).to(io)
        if case["add"]:
            state["residual"] = _hidden(g, tokens, case["width"], std=3.0).to(io)
        state["weight"] = (1.0 + 0.3 * _randn(g, case["width"])).to(io)
    elif op == "gated":
        io = DTYPES[case["io"]]
        heads, dim = case["heads"], case["dim"]
        state["x"] = _randn(g, tokens, heads, dim, std=0.4).to(io)
        # the gate is a column slice of the merged projection's output
        merged = _randn(g, tokens, heads * dim + 4 * dim).to(io)
        state["gate"] = merged[:, 4 * dim:].view(tokens, heads, dim)
        state["weight"] = 1.0 + 0.2 * _randn(g, dim)
    elif op == "quantize":
        state["x"] = _hidden(g, tokens, case["width"]).to(DTYPES[case["io"]])
    else:
        values, scales = _quantize_rows(_hidden(g, tokens, case["k"]))
        state["x"] = (_padded_rows(values), scales.t().contiguous().t())
        state["weight"] = _weight(g, case["n"], case["k"])
    return state


# ------------------------------------------------------------------ one pass

def _run_own(state):
    from logssms_amd.kernel import fp8, norm
    case = state["case"]
    op = case["op"]
    if op == "norm":
        x, weight = state["x"], state["weight"]
        if not case["fp8"]:
            return norm.add_rms_norm(x, state["residual"], weight, EPS) if case["add"] else norm.rms_norm(x, weight, EPS)
        if case["add"]:
            return norm.add_rms_norm_fp8(x, state["residual"], weight, EPS, keep=case["keep"])
        return norm.rms_norm_fp8(x, weight, EPS, keep=case["keep"])
    if op == "gated":
        return norm.rms_norm_gated_fp8(state["x"], state["gate"], state["weight"], EPS)
    if op == "quantize":
        return fp8.quantize_fp8(state["x"])
    return fp8.fp8_linear(fp8.Fp8Tensor(*state["x"]), fp8.Fp8Tensor(*state["weight"]), DTYPES[case["out"]])


def _spread_rows(scales, width):
    return scales.repeat_interleave(BLOCK, 1)[:, :width]


def run(state):
    """One call: the outputs in the order in which the operator returns them
    (the quantised pair first, then the normalised rows in the io type where
    they are kept, then the sum that the next residual is)."""
    if own:
        return _run_own(state)
    case = state["case"]
    op = case["op"]
    if op == "norm":
        io = DTYPES[case["io"]]
        h = state["x"].float()
        if case["add"]:
            h = h + state["residual"].float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * state["weight"].float()
        out = []
        if case["fp8"]:
            out.append(_quantize_rows(y))
        if case["keep"]:
            out.append(y.to(io))
        if case["add"]:
            out.append(h.to(io))
        return out if len(out) > 1 else out[0]
    if op == "gated":
        x, z = state["x"].float(), state["gate"].float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * state["weight"] * (z / (1.0 + torch.exp(-z)))
        return _quantize_rows(y.reshape(y.shape[0], -1))
    if op == "quantize":
        return _quantize_rows(state["x"].float())
    values, scales = state["x"]
    weight, weight_scales = state["weight"]
    n, k = weight.shape
    x = values.float() * _spread_rows(scales, k)
    w = weight.float() * _spread_rows(weight_scales.repeat_interleave(BLOCK, 0)[:n], k)
    return (x @ w.t()).to(DTYPES[case["out"]])


def work(case):
    """Inputs read once and outputs written once; operations of the sums,
    products and roundings of the definition."""
    op, t = case["op"], case["tokens"]
    if op == "linear":
        n, k = case["n"], case["k"]
        kb = -(-k // BLOCK)
        return {"bytes": t * k + 4 * t * kb + n * k + 4 * kb * -(-n // BLOCK) + 2 * t * n, "flops": 2 * t * n * k}
    if op == "gated":
        width = case["heads"] * case["dim"]
        return {"bytes": t * (4 * width + width + 4 * -(-width // BLOCK)) + 4 * case["dim"], "flops": 12 * t * width}
    width = case["width"]
    quantised = width + 4 * -(-width // BLOCK)
    if op == "quantize":
        return {"bytes": t * (2 * width + quantised), "flops": 3 * t * width}
    per_row = 2 * width + 4 * width * case["add"] + quantised * case["fp8"] + 2 * width * case["keep"]
    return {"bytes": t * per_row + 2 * width, "flops": t * width * (4 + case["add"] + 3 * case["fp8"])}


# ------------------------------------------------------------------ 64 bits

def _blocks64(y):
    """value / scale before its rounding to 8 bits, and the scales."""
    rows, width = y.shape
    parts = torch.split(y, BLOCK, dim=1)
    scales = torch.stack([p.abs().max(dim=1).values for p in parts], 1).div(TOP).clamp(min=TINY)
    return torch.cat([p / scales[:, i:i + 1] for i, p in enumerate(parts)], 1), scales


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = state["x"].to(torch.float64)
        if case["add"]:
            h = h + state["residual"].to(torch.float64)
        size = torch.sqrt(torch.sum(h ** 2, dim=1) / case["width"] + EPS)
        y = torch.div(h, size[:, None]) * state["weight"].to(torch.float64)
        out = ([_blocks64(y)] if case["fp8"] else []) + ([y] if case["keep"] else []) + ([h] if case["add"] else [])
        return out if len(out) > 1 else out[0]
    if op == "gated":
        x, z = state["x"].to(torch.float64), state["gate"].to(torch.float64)
        size = torch.sqrt(torch.sum(x ** 2, dim=2) / case["dim"] + EPS)
        y = x / size[:, :, None] * state["weight"].to(torch.float64) * z * torch.sigmoid(z)
        return _blocks64(y.flatten(1))
    if op == "quantize":
        return _blocks64(state["x"].to(torch.float64))
    (values, scales), (weight, weight_scales) = state["x"], state["weight"]
    total = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device=DEV)
    of_column = torch.arange(case["n"], device=DEV) // BLOCK
    for b in range(scales.shape[1]):  # block by block of the summed axis, as the scales are defined
        part = slice(b * BLOCK, min(case["k"], (b + 1) * BLOCK))
        dot = values[:, part].to(torch.float64) @ weight[:, part].to(torch.float64).t()
        total += dot * scales[:, b, None].to(torch.float64) * weight_scales[of_column, b].to(torch.float64)
    return total
