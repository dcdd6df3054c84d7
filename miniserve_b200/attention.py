"""Single-token attention of a batch over a paged cache whose rows share a
prefix: ``prefix_attention``.

The rows of a decode batch often start with the same text (a system prompt, a
schema, a document).  Its keys and values lie in pages that all rows share and
are read once for the whole batch; each row then sees its own pages.  Without
a prefix this is plain paged decode attention.  ``miniserve_b200.kvcache``
describes and writes the cache.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

from . import _lib
from .kvcache import check_cache, check_tensor, half_dtype
from .sampler import _torch

MAX_HEAD_DIM = 128


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
    A row that sees no key has out 0 and lse -inf; so has a row flagged
    MS_ROW_BAD_LENGTH or MS_ROW_BAD_PAGE.
    """
    torch = _torch()
    num_pages, page_size, kv_heads, head_dim = check_cache(cache_k, cache_v)
    dtype, dev = cache_k.dtype, cache_k.device
    check_tensor("q", q, 3, dtype, dev)
    B, heads = q.shape[0], q.shape[1]
    if q.shape[2] != head_dim or heads < 1 or heads % kv_heads:
        raise ValueError(f"q has shape {tuple(q.shape)}: expected [B, a multiple of {kv_heads}, {head_dim}]")
    check_tensor("pages", pages, 2, torch.int32, dev)
    check_tensor("lengths", lengths, 1, torch.int32, dev)
    if pages.shape[0] != B or lengths.shape[0] != B:
        raise ValueError(f"pages has {pages.shape[0]} rows and lengths {lengths.shape[0]} entries, expected {B}")
    if head_dim % 8 or head_dim > MAX_HEAD_DIM:
        raise ValueError(f"head_dim {head_dim} is not a multiple of 8 up to {MAX_HEAD_DIM}")
    for name, t in (("cache_k", cache_k), ("cache_v", cache_v)):
        if t.data_ptr() % 16 or any(n > 1 and s % 8 for n, s in zip(t.shape[:3], t.stride()[:3])):
            raise ValueError(f"{name}'s heads must start 16-byte aligned")
    prefix_length = int(prefix_length)
    if prefix_length < 0:
        raise ValueError("prefix_length must not be negative")
    if prefix_pages is not None:
        check_tensor("prefix_pages", prefix_pages, 1, torch.int32, dev)
    if prefix_length > (0 if prefix_pages is None else prefix_pages.shape[0]) * page_size:
        raise ValueError(f"prefix_pages holds fewer than {prefix_length} keys")
    if scale is None:
        scale = head_dim ** -0.5
    if not (0.0 < scale and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if out is None:
        out = torch.empty((B, heads, head_dim), dtype=dtype, device=dev)
    else:
        check_tensor("out", out, 3, dtype, dev)
        if out.shape != q.shape or any(n > 1 and s <= 0 for n, s in zip(out.shape, out.stride())):
            raise ValueError(f"out must be a {list(q.shape)} tensor that does not repeat its memory")
    lse = torch.empty((B, heads), dtype=torch.float32, device=dev)
    status = torch.empty(B, dtype=torch.int32, device=dev)
    L = _lib.lib()
    a = _lib.PrefixAttentionArgs()
    a.dtype, a.heads, a.kv_heads, a.head_dim, a.rows = half_dtype(cache_k), heads, kv_heads, head_dim, B
    a.q, a.q_row, a.q_head = q.data_ptr(), q.stride(0), q.stride(1)
    # a dimension of one entry is never stepped along: its stride may be anything
    kp, kt, kh = (s if n > 1 else 0 for n, s in zip(cache_k.shape[:3], cache_k.stride()[:3]))
    vp, vt, vh = (s if n > 1 else 0 for n, s in zip(cache_v.shape[:3], cache_v.stride()[:3]))
    a.cache_k, a.ck_page, a.ck_token, a.ck_head = cache_k.data_ptr(), kp, kt, kh
    a.cache_v, a.cv_page, a.cv_token, a.cv_head = cache_v.data_ptr(), vp, vt, vh
    a.pages, a.page_size = num_pages, page_size
    a.table, a.table_width = pages.data_ptr(), pages.shape[1]
    a.table_row = pages.stride(0) if B > 1 else pages.shape[1]
    a.lengths = lengths.data_ptr()
    a.prefix_pages = None if prefix_pages is None else prefix_pages.data_ptr()
    a.prefix_length, a.scale = prefix_length, scale
    a.out, a.out_row, a.out_head = out.data_ptr(), out.stride(0), out.stride(1)
    a.lse, a.status = lse.data_ptr(), status.data_ptr()
    with torch.cuda.device(dev):
        workspace = torch.empty(L.ms_prefix_attention_workspace(B, heads, kv_heads, head_dim, prefix_length),
                                dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
        rc = L.ms_prefix_attention(ctypes.byref(a), torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, "ms_prefix_attention")
    return out, lse, status
