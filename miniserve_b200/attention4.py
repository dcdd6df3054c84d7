"""Attention of one or several tokens a row over a cache held in 4 bits:
``attention_kv4``.

A decode step has one token a row; a step that verifies drafts has the last
accepted token and the drafted ones, each of which sees the keys before it and
its own.  All of a row's tokens share one pass over its keys, read in 4 bits.
``miniserve_b200.kvcache4`` describes and writes the cache.
"""
from __future__ import annotations

from typing import Optional, Tuple

from . import _lib
from .kvcache4 import KvCache4, _of


def attention_kv4(q, cache: KvCache4, pages, lengths, *, scale: Optional[float] = None,
                  out=None) -> Tuple["object", "object", "object"]:
    """Attention of ``q`` [B, heads, head_dim], one token a row, or [B, T, heads,
    head_dim], T tokens a row (at most 1024), over the cache.

    Token t of row b sees the first ``lengths[b, t]`` keys ([B, T] int32, or [B]
    for one token a row) of the row's pages ``pages[b]`` ([B, width] int32;
    entries past the row's keys are not read).  Drafted tokens that see one
    another in order have lengths ``n - T + 1 .. n``; a token that sees nothing
    (padding) has length 0.  ``scale`` defaults to ``head_dim ** -0.5``.  Query
    heads ``h * heads // kv_heads`` on share key head ``h``.

    Returns ``(out, lse, status)``: q's shape in q's type, the logarithm of the
    softmax's sum in fp32 (q's shape without head_dim), and [B] int32 MS_ROW_*
    bits.  A token that sees no key has out 0 and lse -inf; so have all tokens
    of a row flagged MS_ROW_BAD_LENGTH, and the heads of a row flagged
    MS_ROW_BAD_PAGE that met the page.  What the cache holds past a token's
    keys does not touch its result.  Scores and sums are fp32; weights are
    rounded to fp16 (for fp16 queries to two halves), the result once; entries
    whose 32 share a scale below 2^-20 of the largest value scale of the head's
    keys lose bits.
    """
    entry = _lib.binding()
    try:
        return entry.attention_kv4(*_of(cache), q, pages, lengths, scale, out)
    except entry.CallError as e:
        _lib.check(e.args[0], "ms_kv4_attention")
        raise
