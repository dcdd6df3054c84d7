"""Writing a paged key/value cache: ``rope_table`` and ``append_kv``.

A cache is a pair of tensors [pages, page_size, kv_heads, head_dim] (bf16 or
fp16); the first three dimensions may lie in any order in memory, so a cache
stored head-major is passed as its ``transpose(1, 2)`` view.  Slot ``page *
page_size + offset`` names one token's place in it.  ``append_kv`` writes new
tokens there with the position rotation applied on the way (one launch:
queries, keys and values), for prompts and single decode tokens alike;
``miniserve_b200.attention`` reads what it wrote.
"""
from __future__ import annotations

from typing import Optional, Tuple

from . import _lib
from .sampler import _torch


def rope_table(positions: int, rotary: int, base: float = 10000.0, device="cuda"):
    """[positions, 2, rotary // 2] fp32: the cosines, then the sines, of
    ``p * base ** (-2 i / rotary)``, computed in float64 and rounded once."""
    torch = _torch()
    if positions < 1 or rotary < 2 or rotary % 2:
        raise ValueError("rope_table needs at least one position and an even, positive rotary size")
    inv = float(base) ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], 1).float()


def append_kv(cache_k, cache_v, k, v, slots, *, q=None, positions=None, rope=None, interleaved: bool = False,
              q_out=None) -> Tuple[Optional["object"], "object"]:
    """Write new tokens' keys and values into their cache slots, rotated.

    ``k``, ``v`` [T, kv_heads, head_dim] and optionally ``q`` [T, heads,
    head_dim] are tensors of the cache's type, contiguous in the last dimension
    (slices of a fused projection's output are fine).  ``slots`` [T] int64; a
    negative slot is padding and writes nothing.  ``rope`` is
    ``rope_table(...)`` and ``positions`` [T] int64 its rows: the first
    ``rotary`` entries of every query and key head are rotated, in pairs
    (i, i + rotary/2) or, ``interleaved``, (2i, 2i + 1).  Without ``rope``
    everything is copied.

    Returns ``(q_out, status)``: the rotated queries (``q_out`` if given, which
    may be ``q`` itself; None without ``q``) and [T] int32 MS_ROW_* bits
    (MS_ROW_BAD_SLOT, MS_ROW_BAD_POSITION: nothing was written to the cache).
    """
    entry = _lib.binding()
    try:
        return entry.append_kv(cache_k, cache_v, k, v, slots, q, positions, rope, interleaved, q_out)
    except entry.CallError as e:
        _lib.check(e.args[0], "ms_kv_append")
        raise
