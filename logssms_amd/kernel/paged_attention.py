"""The full-attention side of a hybrid model's cache: keys and values appended to
its pages (``csrc/rotary.hip``), and the attention that reads them for a batch
whose requests share prefixes (``csrc/paged_attention.hip``).

Caches are ``[pages, page size, kv heads, dim]`` views with unit channel stride,
those of ``HybridBlockPool.kv_cache`` or any others.  A token's place is its
slot, ``page * page size + offset``.

    q = append_paged_kv(k, v, k_cache, v_cache, slots, positions=positions, rotary=rotary, q=q)
    out = paged_attention(q, k_cache, v_cache, page_table, seq_lens, shared_lens=shared_lens)

Both are for inference and record no gradient.
"""

from __future__ import annotations

import torch

from .. import _lib
from .rotary import Rotary


def append_paged_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    slots: torch.Tensor, *, positions: torch.Tensor | None = None, rotary: Rotary | None = None,
                    q: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """``k`` and ``v`` [tokens, kv heads, dim] to the slots [tokens] (int32 or int64,
    no two alike) of the caches, which may not overlap, ``k`` rotated by ``positions``
    where a ``rotary`` is given.  A slot below 0, or past the cache, takes no write.
    ``q`` [tokens, heads, dim] is rotated in the same launch and returned (``q_out``,
    which may be ``q`` itself, or a new tensor).  fp32, bf16 or f16, one dtype for all."""
    turns, interleaved, scale = (None, False, 1.0) if rotary is None else rotary
    return _lib.host().append_paged_kv(k, v, k_cache, v_cache, slots, positions, turns, interleaved, scale, q, q_out)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, *, shared_lens: torch.Tensor | None = None,
                    group_offsets: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False
                    ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of ``q`` [tokens, heads, dim] (bf16 or f16, dim 64, 128 or
    256) over a paged cache, heads of queries in equal groups to each key head.

    Request r owns the tokens ``cu_seqlens[r]`` .. ``cu_seqlens[r + 1] - 1``, without
    ``cu_seqlens`` token r: the last ones of its ``seq_lens[r]`` positions, whose keys
    are in the cache already.  Position p lies in page ``page_table[r, p // page
    size]`` (a page outside of the cache stands for zeros).  ``scale`` is
    ``dim ** -0.5`` by default.

    The requests ``group_offsets[g]`` .. ``group_offsets[g + 1] - 1`` of group g (all of
    them without ``group_offsets``) share their first ``shared_lens[g]`` positions: the
    same pages in each of their rows, of which the first request's is read (an empty
    request's too).  These are attended once for the group, and nothing else depends on
    it.

    A token that sees no position gives zeros, one all of whose scores are -inf NaN;
    tokens that no request owns are left as they were in ``out`` (a new one holds
    anything there).  ``return_lse``: also the logarithm of each row's sum of exponentials,
    fp32 [tokens, heads], -inf where nothing is seen.  Lengths, offsets and tables are read
    on the device: a captured call follows them at each replay."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    result, lse = _lib.host().paged_attention(q, k_cache, v_cache, page_table, seq_lens, shared_lens, group_offsets,
                                              cu_seqlens, scale, out, return_lse)
    return (result, lse) if return_lse else result


__all__ = ["append_paged_kv", "paged_attention"]
