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

import ctypes
from typing import Optional, Tuple

from . import _lib
from ._launch import launch, refuse
from .sampler import _torch


def half_dtype(t) -> int:
    """The library's code of a bf16 or fp16 tensor's type."""
    torch = _torch()
    if t.dtype is torch.bfloat16:
        return _lib.MS_DTYPE_BF16
    if t.dtype is torch.float16:
        return _lib.MS_DTYPE_F16
    raise TypeError(f"dtype {t.dtype} is not bfloat16 or float16")


def check_cache(cache_k, cache_v):
    """(shape, K's strides, V's strides) of a cache, after the checks the
    kernels rely on."""
    torch = _torch()
    if not isinstance(cache_k, torch.Tensor) or not cache_k.is_cuda:
        raise TypeError("cache_k must be a CUDA tensor")
    shape, sk = cache_k.shape, cache_k.stride()
    if not isinstance(cache_v, torch.Tensor) or cache_v.dtype is not cache_k.dtype \
            or cache_v.device != cache_k.device or cache_v.shape != shape or len(shape) != 4 or 0 in shape \
            or sk[3] != 1 or cache_v.stride(3) != 1:
        refuse("cache_k", cache_k, (None,) * 4, cache_k.dtype, cache_k.device)
        refuse("cache_v", cache_v, tuple(shape), cache_k.dtype, cache_k.device)
        if 0 in shape:
            raise ValueError("the cache must be a non-empty [pages, page_size, kv_heads, head_dim] tensor")
    sv = cache_v.stride()
    if min(sk) <= 0 or min(sv) <= 0:
        for name, st in (("cache_k", sk), ("cache_v", sv)):
            if any(n > 1 and s <= 0 for n, s in zip(shape, st)):
                raise ValueError(f"{name} must not repeat its memory (an expanded tensor)")
    return shape, sk, sv


def heads_of(name: str, t, tokens: int, heads: Optional[int], head_dim: int, dtype, device):
    """(pointer, token stride, head stride) of a [tokens, heads, head_dim]
    tensor, contiguous in its heads' entries."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.dim() != 3 \
            or t.shape != (tokens, t.shape[1] if heads is None else heads, head_dim) or t.stride(2) != 1:
        refuse(name, t, (tokens, heads, head_dim), dtype, device)
    st = t.stride()
    return t.data_ptr(), st[0], st[1]


def vector_of(name: str, t, n: int, dtype, device) -> int:
    """Pointer of a contiguous [n] tensor."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != (n,) \
            or t.stride(0) != 1:
        refuse(name, t, (n,), dtype, device)
    return t.data_ptr()


def check_writable(name: str, t) -> None:
    st = t.stride()
    if min(st) <= 0 and any(n > 1 and s <= 0 for n, s in zip(t.shape, st)):
        raise ValueError(f"{name} must not repeat its memory (an expanded tensor)")


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
    torch = _torch()
    shape, sk, sv = check_cache(cache_k, cache_v)
    pages, page_size, kv_heads, head_dim = shape
    dtype, dev = cache_k.dtype, cache_k.device
    a = _lib.KvAppendArgs()
    a.dtype = half_dtype(cache_k)
    T = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else 0
    a.k, a.k_token, a.k_head = heads_of("k", k, T, kv_heads, head_dim, dtype, dev)
    a.v, a.v_token, a.v_head = heads_of("v", v, T, kv_heads, head_dim, dtype, dev)
    a.slots = vector_of("slots", slots, T, torch.int64, dev)
    a.kv_heads, a.head_dim, a.tokens = kv_heads, head_dim, T
    a.interleaved = 1 if interleaved else 0
    if rope is not None:
        if not isinstance(rope, torch.Tensor) or rope.dtype is not torch.float32 or rope.device != dev \
                or rope.dim() != 3 or rope.shape[1] != 2 or not rope.is_contiguous():
            refuse("rope", rope, (None, 2, None), torch.float32, dev)
            raise ValueError("rope must be a contiguous [positions, 2, rotary / 2] table (rope_table)")
        rows, _, half = rope.shape
        if rows < 1 or not 0 < 2 * half <= head_dim:
            raise ValueError(f"rope rotates {2 * half} entries of heads of {head_dim}, at {rows} positions")
        if positions is None:
            raise ValueError("rope needs positions")
        a.positions = vector_of("positions", positions, T, torch.int64, dev)
        a.rotary, a.table, a.table_rows = 2 * half, rope.data_ptr(), rows
    if q is not None:
        a.q, a.q_token, a.q_head = heads_of("q", q, T, None, head_dim, dtype, dev)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=dtype, device=dev)
        elif q_out.data_ptr() == a.q and q_out.stride() != q.stride():
            raise ValueError("q_out in place of q must have q's strides")
        a.heads = q.shape[1]
        a.q_out, a.q_out_token, a.q_out_head = heads_of("q_out", q_out, T, a.heads, head_dim, dtype, dev)
        check_writable("q_out", q_out)
    elif q_out is not None:
        raise ValueError("q_out needs q")
    status = torch.empty(T, dtype=torch.int32, device=dev)
    a.cache_k, a.ck_page, a.ck_token, a.ck_head = cache_k.data_ptr(), sk[0], sk[1], sk[2]
    a.cache_v, a.cv_page, a.cv_token, a.cv_head = cache_v.data_ptr(), sv[0], sv[1], sv[2]
    a.pages, a.page_size, a.status = pages, page_size, status.data_ptr()
    rc = launch(dev, _lib.lib().ms_kv_append, ctypes.byref(a))
    if rc:
        _lib.check(rc, "ms_kv_append")
    return q_out, status
