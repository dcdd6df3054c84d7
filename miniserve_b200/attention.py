"""Single-token attention of a batch over a paged cache whose rows share a
prefix: ``prefix_attention``.

The rows of a decode batch often start with the same text (a system prompt, a
schema, a document).  Its keys and values lie in pages that all rows share and
are read once for the whole batch; each row then sees its own pages.  Without
a prefix this is plain paged decode attention.  ``miniserve_b200.kvcache``
describes and writes the cache.
"""
from __future__ import annotations

from typing import Optional, Tuple

from . import _lib


def prefix_attention(q, cache_k, cache_v, pages, lengths, *, prefix_pages=None, prefix_length: int = 0,
                     scale: Optional[float] = None, out=None) -> Tuple["object", "object", "object"]:
    """Attention of ``q`` [B, heads, head_dim], one token a row, over the cache.

    Row b sees the first ``prefix_length`` keys of ``prefix_pages`` ([n] int32,
    shared by all rows) and the first ``lengths[b]`` ([B] int32) keys of its
    own pages ``pages[b]`` ([B, width] int32; entries past the row's keys are
    not read).  ``scale`` defaults to ``head_dim ** -0.5``.  Query heads
    ``h * heads // kv_heads`` on share key head ``h``.

    Returns ``(out, lse, status)``: [B, heads, head_dim] in q's type, the
    logarithm of the softmax's sum [B, heads] fp32, and [B] int32 MS_ROW_* bits.
    Heads are up to 128 entries, a multiple of 8, and start 16-byte aligned.
    A row that sees no key has out 0 and lse -inf; so has a row flagged
    MS_ROW_BAD_LENGTH or MS_ROW_BAD_PAGE, and the heads of a row flagged
    MS_ROW_WAIT_TIMEOUT that lost a part of the prefix (a wait inside its kernel
    was given up after 1 s).
    """
    entry = _lib.binding()
    try:
        return entry.prefix_attention(q, cache_k, cache_v, pages, lengths, prefix_pages, prefix_length, scale, out)
    except entry.CallError as e:
        _lib.check(e.args[0], "ms_prefix_attention")
        raise
