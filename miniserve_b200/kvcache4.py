"""A paged key/value cache held in 4 bits: ``KvCache4``, ``append_kv4`` and
``read_kv4``.

Every 32 entries of a head share a scale and a middle (fp16) and are held as
4-bit codes: 5 bits an entry instead of the 16 of ``miniserve_b200.kvcache``'s
caches, so that a decode step reads less than a third of the bytes and the same
memory holds three times the tokens.  ``append_kv4`` quantises new tokens as it
writes them, the position rotation applied on the way; ``read_kv4`` gives back
what the cache stands for, in the model's type;
``miniserve_b200.attention4`` attends over the codes as they are.  Slots are
those of ``append_kv``: ``page * page_size + offset``.
"""
from __future__ import annotations

from typing import Optional, Tuple

from . import _lib
from .sampler import _torch

GROUP = 32  # entries that share a scale and a middle


def _stored(head_dim: int) -> Tuple[int, int]:
    """(bytes of codes, pairs of parameters) of a stored head."""
    used = max(2, -(-head_dim // GROUP))
    return used * GROUP // 2, 4 if used == 3 else used


class KvCache4:
    """The four tensors of a 4-bit cache.

    ``k_codes``, ``v_codes`` uint8 [pages, kv_heads, page_size, padded / 2]
    (``padded``: head_dim rounded up to a multiple of 32, at least 64; byte j
    holds entries 2j, in its low four bits, and 2j + 1) and ``k_params``,
    ``v_params`` fp16 [pages, kv_heads, page_size, groups, 2], the scale and the
    middle of every 32 entries (``groups``: 2 or 4, as many as padded needs).
    Entry i stands for ``middle + scale * (code - 8)``.  All are contiguous
    and start aligned: codes to 16 bytes, parameters to a slot's (8 for two
    groups, 16 for four).  A range of pages (``cache[first:last]``) is a cache
    too.

    ``dtype`` (bfloat16 or float16) is the model's type: what ``append_kv4``
    takes and ``read_kv4`` gives.  ``head_dim`` is a multiple of 16 up to 128.
    """

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params", "head_dim", "dtype", "_args")

    def __init__(self, k_codes, k_params, v_codes, v_params, *, head_dim: int, dtype) -> None:
        torch = _torch()
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"dtype {dtype} is not bfloat16 or float16")
        if not isinstance(head_dim, int) or head_dim < 16 or head_dim % 16 or head_dim > 128:
            raise ValueError(f"head_dim {head_dim!r} is not a multiple of 16 up to 128")
        row, groups = _stored(head_dim)
        for name, t, kind, tail in (("k_codes", k_codes, torch.uint8, (row,)), ("k_params", k_params, torch.float16, (groups, 2)),
                                    ("v_codes", v_codes, torch.uint8, (row,)), ("v_params", v_params, torch.float16, (groups, 2))):
            if not isinstance(t, torch.Tensor) or t.dtype != kind:
                raise TypeError(f"{name} must be a {kind} tensor")
            if t.dim() != 3 + len(tail) or tuple(t.shape[3:]) != tail or t.shape[:3] != k_codes.shape[:3]:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected [pages, kv_heads, page_size, "
                                 f"{', '.join(map(str, tail))}]")
            if t.device != k_codes.device:
                raise ValueError(f"{name} is on {t.device}, k_codes on {k_codes.device}")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            align = groups * 4 if kind == torch.float16 else 16
            if t.data_ptr() % align:
                raise ValueError(f"{name} must start {align}-byte aligned")
        if not k_codes.numel():
            raise ValueError("the cache is empty")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.head_dim, self.dtype = head_dim, dtype
        self._args = (k_codes, k_params, v_codes, v_params, head_dim, dtype)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype=None, device="cuda") -> "KvCache4":
        """A cache of zeros: ``pages`` pages of ``page_size`` tokens."""
        torch = _torch()
        if not isinstance(head_dim, int) or head_dim < 16 or head_dim % 16 or head_dim > 128:
            raise ValueError(f"head_dim {head_dim!r} is not a multiple of 16 up to 128")
        row, groups = _stored(head_dim)
        lead = (pages, kv_heads, page_size)
        k_codes, v_codes = (torch.zeros((*lead, row), dtype=torch.uint8, device=device) for _ in range(2))
        k_params, v_params = (torch.zeros((*lead, groups, 2), dtype=torch.float16, device=device) for _ in range(2))
        return cls(k_codes, k_params, v_codes, v_params, head_dim=head_dim, dtype=dtype or torch.bfloat16)

    def __getitem__(self, pages: slice) -> "KvCache4":
        if not isinstance(pages, slice):
            raise TypeError("a cache is indexed by a range of pages")
        return KvCache4(*(t[pages] for t in self._args[:4]), head_dim=self.head_dim, dtype=self.dtype)

    @property
    def pages(self) -> int:
        return self.k_codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def device(self):
        return self.k_codes.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._args[:4])


def _of(cache) -> tuple:
    if not isinstance(cache, KvCache4):
        raise TypeError("cache must be a KvCache4")
    return cache._args


def append_kv4(cache: KvCache4, k, v, slots, *, q=None, positions=None, rope=None, interleaved: bool = False,
               q_out=None) -> Tuple[Optional["object"], "object"]:
    """Write new tokens' keys and values into their cache slots, rotated and
    quantised.

    The arguments are ``append_kv``'s: ``k``, ``v`` [T, kv_heads, head_dim] and
    optionally ``q`` [T, heads, head_dim] of the cache's ``dtype``, ``slots`` [T]
    int64 (a negative slot is padding and writes nothing), ``rope`` a
    ``rope_table`` and ``positions`` [T] int64 its rows.  Slots of one call must
    differ: of two equal ones the slot may hold some of either token's entries.

    A group of 32 entries (of the rotated key, which is not rounded in between)
    is held to half its scale, (max - min) / 30, and the fp16 roundings of scale
    and middle.  Entries of magnitudes past fp16's range, infinities and NaN are
    not held: their groups read back as NaN and the token is flagged
    MS_ROW_NONFINITE.

    Returns ``(q_out, status)``: the rotated queries in 16 bits (``q_out`` if
    given, which may be ``q`` itself; None without ``q``) and [T] int32 MS_ROW_*
    bits (MS_ROW_BAD_SLOT, MS_ROW_BAD_POSITION: nothing was written to the
    cache; MS_ROW_NONFINITE).
    """
    entry = _lib.binding()
    try:
        return entry.append_kv4(*_of(cache), k, v, slots, q, positions, rope, interleaved, q_out)
    except entry.CallError as e:
        _lib.check(e.args[0], "ms_kv4_append")
        raise


def read_kv4(cache: KvCache4, slots, *, k_out=None, v_out=None) -> Tuple["object", "object", "object"]:
    """What the cache stands for in ``slots`` [T] int64.

    Returns ``(k, v, status)``: [T, kv_heads, head_dim] each in the cache's
    ``dtype`` (``k_out`` and ``v_out`` if given), computed in fp32 and rounded
    once (entries past fp16's range become its largest), and [T] int32 MS_ROW_*
    bits.  A negative slot (padding) reads as zeros, and so does one past the
    cache, which is flagged MS_ROW_BAD_SLOT.
    """
    entry = _lib.binding()
    try:
        return entry.read_kv4(*_of(cache), slots, k_out, v_out)
    except entry.CallError as e:
        _lib.check(e.args[0], "ms_kv4_read")
        raise
