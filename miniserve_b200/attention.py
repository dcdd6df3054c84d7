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
import functools
import math
from typing import Optional, Tuple

from . import _lib
from ._launch import launch, refuse
from .kvcache import check_cache, check_writable, half_dtype, heads_of, vector_of
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
    shape, sk, sv = check_cache(cache_k, cache_v)
    num_pages, page_size, kv_heads, head_dim = shape
    dtype, dev = cache_k.dtype, cache_k.device
    a = _lib.PrefixAttentionArgs()
    a.dtype = half_dtype(cache_k)
    B = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
    a.q, a.q_row, a.q_head = heads_of("q", q, B, None, head_dim, dtype, dev)
    heads = q.shape[1]
    if heads < 1 or heads % kv_heads:
        raise ValueError(f"q has {heads} heads, expected a multiple of the cache's {kv_heads}")
    if not isinstance(pages, torch.Tensor) or pages.dtype is not torch.int32 or pages.device != dev \
            or pages.dim() != 2 or pages.shape[0] != B or pages.stride(1) != 1:
        refuse("pages", pages, (B, None), torch.int32, dev)
    a.lengths = vector_of("lengths", lengths, B, torch.int32, dev)
    if head_dim % 8 or head_dim > MAX_HEAD_DIM:
        raise ValueError(f"head_dim {head_dim} is not a multiple of 8 up to {MAX_HEAD_DIM}")
    a.cache_k, a.ck_page, a.ck_token, a.ck_head = cache_k.data_ptr(), sk[0], sk[1], sk[2]
    a.cache_v, a.cv_page, a.cv_token, a.cv_head = cache_v.data_ptr(), sv[0], sv[1], sv[2]
    if (sk[0] | sk[1] | sk[2] | sv[0] | sv[1] | sv[2]) & 7 or (a.cache_k | a.cache_v) & 15:
        # a dimension of one entry is never stepped along: its stride may be anything
        kp, kt, kh = (s if n > 1 else 0 for n, s in zip(shape, sk[:3]))
        vp, vt, vh = (s if n > 1 else 0 for n, s in zip(shape, sv[:3]))
        if (kp | kt | kh | vp | vt | vh) & 7 or (a.cache_k | a.cache_v) & 15:
            raise ValueError("the cache's heads must start 16-byte aligned")
        a.ck_page, a.ck_token, a.ck_head, a.cv_page, a.cv_token, a.cv_head = kp, kt, kh, vp, vt, vh
    prefix_length = int(prefix_length)
    if prefix_pages is not None:
        a.prefix_pages = vector_of("prefix_pages", prefix_pages, prefix_pages.shape[0], torch.int32, dev)
    if not 0 <= prefix_length <= (0 if prefix_pages is None else prefix_pages.shape[0]) * page_size:
        raise ValueError(f"prefix_length {prefix_length} does not fit prefix_pages")
    if scale is None:
        scale = head_dim ** -0.5
    elif not (0.0 < scale and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if out is None:
        out = torch.empty((B, heads, head_dim), dtype=dtype, device=dev)
    a.out, a.out_row, a.out_head = heads_of("out", out, B, heads, head_dim, dtype, dev)
    check_writable("out", out)
    lse = torch.empty((B, heads), dtype=torch.float32, device=dev)
    status = torch.empty(B, dtype=torch.int32, device=dev)
    bytes_needed = _workspace(B, heads, kv_heads, head_dim, prefix_length, dev.index)
    workspace = torch.empty(bytes_needed, dtype=torch.uint8, device=dev)
    a.heads, a.kv_heads, a.head_dim, a.rows = heads, kv_heads, head_dim, B
    a.pages, a.page_size = num_pages, page_size
    a.table, a.table_width = pages.data_ptr(), pages.shape[1]
    a.table_row = pages.stride(0) if B > 1 else a.table_width
    a.prefix_length, a.scale = prefix_length, scale
    a.lse, a.status = lse.data_ptr(), status.data_ptr()
    a.workspace, a.workspace_bytes = workspace.data_ptr(), bytes_needed
    rc = launch(dev, _lib.lib().ms_prefix_attention, ctypes.byref(a))
    if rc:
        _lib.check(rc, "ms_prefix_attention")
    return out, lse, status


@functools.lru_cache(maxsize=4096)
def _workspace(rows: int, heads: int, kv_heads: int, head_dim: int, prefix_length: int, device: int) -> int:
    """Bytes of a call's workspace: a function of its sizes and the device alone."""
    with _torch().cuda.device(device):
        return _lib.lib().ms_prefix_attention_workspace(rows, heads, kv_heads, head_dim, prefix_length)
