"""Rotary positions on the gfx950 kernel ``gdn_apply_rotary`` (``csrc/rotary.hip``):
half and interleaved layouts, all of a head or its first part, plain frequencies
or ones stretched for long contexts.

    rotary = rotary_embedding(64, 1e7, device="cuda")   # once, with the model
    q, k = apply_rotary(q, k, positions, rotary)        # [tokens, heads, dim]

Angles are products of the position itself in 64 bits: there is no table, and
positions up to some 2^30 cost no precision in fp32 (at 2^40 the fastest pair is off by
10^-4 radians).  ``append_paged_kv`` does the same on the way to the cache.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _lib


class Rotary(NamedTuple):
    """``turns`` float64 [rotated / 2]: revolutions per position of each pair,
    ``(x[i], x[i + rotated / 2])`` or, ``interleaved``, ``(x[2i], x[2i + 1])``;
    ``scale``: a factor on the rotated values."""

    turns: torch.Tensor
    interleaved: bool = False
    scale: float = 1.0

    @property
    def rotated(self) -> int:
        """The channels of a head that are rotated, its first ones."""
        return 2 * self.turns.numel()


SCALINGS = ("none", "linear", "base", "wavelength", "yarn")


def rotary_embedding(rotated: int, base: float = 10000.0, *, interleaved: bool = False, scaling: str = "none",
                     factor: float = 1.0, original_length: int | None = None, slow: float = 1.0,
                     fast: float | None = None, scale: float | None = None, device=None) -> Rotary:
    """Pair i turns by ``base ** (-2 i / rotated)`` radians a position, stretched
    by ``factor`` for contexts beyond ``original_length``:

    * ``"linear"``: every angle divided by ``factor``;
    * ``"base"``: the base times ``factor ** (rotated / (rotated - 2))``, so that
      the slowest pair is stretched by ``factor`` and the fastest not at all;
    * ``"wavelength"``: pairs with at least ``fast`` (4) rotations over the original
      length stay, those with at most ``slow`` (1) are divided by ``factor``, linearly
      in their rotations between;
    * ``"yarn"``: the same with ``fast`` 32, linearly in the pair's index between the
      whole indices around both bounds, and a ``scale`` of ``0.1 ln(factor) + 1``.

    ``scale`` overrides the factor on the rotated values."""
    assert rotated >= 0 and rotated % 2 == 0, "an even number of rotated channels"
    assert base > 0 and factor > 0, "base and factor must be positive"
    assert scaling in SCALINGS, f"scaling must be one of {SCALINGS}"
    assert scaling not in ("wavelength", "yarn") or (original_length is not None and original_length > 0), \
        "original_length is needed"
    if scaling == "none":
        assert factor == 1.0, "a factor without a scaling"
    if scaling == "base":
        base = base * factor ** (rotated / max(rotated - 2, 1))
    index = torch.arange(rotated // 2, dtype=torch.float64)
    turns = base ** (-2 * index / max(rotated, 1)) / (2 * math.pi)
    if scaling == "linear":
        turns = turns / factor
    elif scaling == "wavelength":
        fast = 4.0 if fast is None else fast
        assert fast > slow, "fast must exceed slow"
        kept = ((original_length * turns - slow) / (fast - slow)).clamp(0, 1)
        turns = turns * (kept + (1 - kept) / factor)
    elif scaling == "yarn":
        fast = 32.0 if fast is None else fast
        assert fast > slow > 0 and base != 1, "fast must exceed slow"
        # the (fractional) pair with so many rotations over the original length
        low, high = (rotated * math.log(original_length / (2 * math.pi * n)) / (2 * math.log(base)) for n in (fast, slow))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rotated - 1)
        kept = 1 - ((index - low) / max(high - low, 1e-3)).clamp(0, 1)
        turns = turns * (kept + (1 - kept) / factor)
        if scale is None and factor > 1:
            scale = 0.1 * math.log(factor) + 1.0
    return Rotary(turns.to(device), interleaved, 1.0 if scale is None else float(scale))


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary, *,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``q`` [tokens, heads, dim] (and ``k``, with heads of its own) rotated by
    ``positions`` [tokens] (int32 or int64), fp32, bf16 or f16, computed in fp32
    and rounded once; strided views are read as they are.  ``q_out`` and ``k_out``
    may be the operands themselves, which are then rotated in place."""
    return _lib.host().apply_rotary(q, k, positions, rotary.turns, rotary.interleaved, rotary.scale, q_out, k_out)


__all__ = ["Rotary", "apply_rotary", "rotary_embedding"]
