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
from .sampler import _torch


def half_dtype(t) -> int:
    """The library's code of a bf16 or fp16 tensor's type."""
    torch = _torch()
    if t.dtype == torch.bfloat16:
        return _lib.MS_DTYPE_BF16
    if t.dtype == torch.float16:
        return _lib.MS_DTYPE_F16
    raise TypeError(f"dtype {t.dtype} is not bfloat16 or float16")


def check_tensor(name: str, t, dims: int, dtype, device) -> None:
    """A tensor of the given type on ``device`` with ``dims`` dimensions, the
    last of them contiguous."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dim() != dims:
        raise ValueError(f"{name} has {t.dim()} dimensions, expected {dims}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def check_cache(cache_k, cache_v) -> Tuple[int, int, int, int]:
    """(pages, page_size, kv_heads, head_dim) of a cache, after the checks the
    kernels rely on."""
    torch = _torch()
    if not isinstance(cache_k, torch.Tensor) or not cache_k.is_cuda:
        raise TypeError("cache_k must be a CUDA tensor")
    half_dtype(cache_k)
    for name, t in (("cache_k", cache_k), ("cache_v", cache_v)):
        check_tensor(name, t, 4, cache_k.dtype, cache_k.device)
        if 0 in t.shape:
            raise ValueError(f"{name} must be a non-empty [pages, page_size, kv_heads, head_dim] tensor")
        if any(n > 1 and s <= 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{name} must not repeat its memory (an expanded tensor)")
    if cache_v.shape != cache_k.shape:
        raise ValueError(f"cache_v has shape {tuple(cache_v.shape)}, cache_k {tuple(cache_k.shape)}")
    return tuple(cache_k.shape)


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
    pages, page_size, kv_heads, head_dim = check_cache(cache_k, cache_v)
    dtype, dev = cache_k.dtype, cache_k.device
    check_tensor("k", k, 3, dtype, dev)
    check_tensor("v", v, 3, dtype, dev)
    T = k.shape[0]
    for name, t in (("k", k), ("v", v)):
        if t.shape != (T, kv_heads, head_dim):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({T}, {kv_heads}, {head_dim})")
    check_tensor("slots", slots, 1, torch.int64, dev)
    if slots.shape[0] != T:
        raise ValueError(f"slots has {slots.shape[0]} entries, expected {T}")
    a = _lib.KvAppendArgs()
    a.dtype, a.kv_heads, a.head_dim, a.tokens = half_dtype(cache_k), kv_heads, head_dim, T
    a.interleaved = int(bool(interleaved))
    if rope is not None:
        check_tensor("rope", rope, 3, torch.float32, dev)
        if rope.shape[1] != 2 or rope.shape[0] < 1 or not rope.is_contiguous():
            raise ValueError("rope must be a contiguous [positions, 2, rotary / 2] table (rope_table)")
        a.rotary = 2 * rope.shape[2]
        if not 0 < a.rotary <= head_dim:
            raise ValueError(f"rope rotates {a.rotary} entries, the heads have {head_dim}")
        if positions is None:
            raise ValueError("rope needs positions")
        check_tensor("positions", positions, 1, torch.int64, dev)
        if positions.shape[0] != T:
            raise ValueError(f"positions has {positions.shape[0]} entries, expected {T}")
        a.positions, a.table, a.table_rows = positions.data_ptr(), rope.data_ptr(), rope.shape[0]
    if q is not None:
        check_tensor("q", q, 3, dtype, dev)
        if q.shape[0] != T or q.shape[2] != head_dim:
            raise ValueError(f"q has shape {tuple(q.shape)}, expected ({T}, heads, {head_dim})")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=dtype, device=dev)
        else:
            check_tensor("q_out", q_out, 3, dtype, dev)
            if q_out.shape != q.shape:
                raise ValueError(f"q_out has shape {tuple(q_out.shape)}, expected {tuple(q.shape)}")
            if any(n > 1 and st <= 0 for n, st in zip(q_out.shape, q_out.stride())):
                raise ValueError("q_out must not repeat its memory (an expanded tensor)")
            if q_out.data_ptr() == q.data_ptr() and q_out.stride() != q.stride():
                raise ValueError("q_out in place of q must have q's strides")
        a.heads = q.shape[1]
        a.q, a.q_token, a.q_head = q.data_ptr(), q.stride(0), q.stride(1)
        a.q_out, a.q_out_token, a.q_out_head = q_out.data_ptr(), q_out.stride(0), q_out.stride(1)
    elif q_out is not None:
        raise ValueError("q_out needs q")
    status = torch.empty(T, dtype=torch.int32, device=dev)
    a.k, a.k_token, a.k_head = k.data_ptr(), k.stride(0), k.stride(1)
    a.v, a.v_token, a.v_head = v.data_ptr(), v.stride(0), v.stride(1)
    a.cache_k, (a.ck_page, a.ck_token, a.ck_head) = cache_k.data_ptr(), cache_k.stride()[:3]
    a.cache_v, (a.cv_page, a.cv_token, a.cv_head) = cache_v.data_ptr(), cache_v.stride()[:3]
    a.pages, a.page_size, a.slots, a.status = pages, page_size, slots.data_ptr(), status.data_ptr()
    with torch.cuda.device(dev):
        rc = _lib.lib().ms_kv_append(ctypes.byref(a), torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, "ms_kv_append")
    return q_out, status
