"""8-bit integer product with a scale for each token and each output channel:
``quantize_rows``, ``int8_matmul`` and the layer ``Int8Linear``.

    head = Int8Linear.from_float(lm_head_weight)        # [V, K], once
    logits = head(hidden)                               # [B, V] fp32
    tokens, probs, status = Sampler().sample_batch(logits, ...)

A token's integers are its entries over scale = max |x| / 127, rounded to the
nearest (ties to even); the integer sums are exact and scaled in fp32.  A row
with a NaN or an infinity gives NaN outputs.
"""
from __future__ import annotations

from typing import Optional, Tuple

from . import _lib
from ._launch import launch
from .sampler import _torch

MAX_INNER = 131072  # the int32 sum of 127 * 127 * K stays exact


def _dtype_code(dtype) -> int:
    torch = _torch()
    if dtype is torch.float32:
        return _lib.MS_DTYPE_F32
    if dtype is torch.bfloat16:
        return _lib.MS_DTYPE_BF16
    if dtype is torch.float16:
        return _lib.MS_DTYPE_F16
    raise TypeError(f"dtype {dtype} is not float32, bfloat16 or float16")


def _matrix(name: str, t, dtype=None):
    """A CUDA matrix, contiguous in its rows."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.dim() != 2 or t.shape[1] < 1:
        raise ValueError(f"{name} must be a [rows, entries] matrix")
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name} must have contiguous rows that do not overlap")
    return t


def _pitch(t) -> int:
    """Row stride of a checked matrix (a single row's may be anything)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _vector(name: str, t, n: int, device):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
        raise TypeError(f"{name} must be a float32 tensor")
    if t.device != device or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] tensor on {device}")
    return t


def _check_inner(K: int) -> None:
    if K > MAX_INNER:
        raise ValueError(f"rows of {K} entries: the integer sum is exact up to {MAX_INNER}")


def _empty_rows(M: int, K: int, device):
    """[M, K] int8 whose rows lie a multiple of 16 bytes apart."""
    torch = _torch()
    return torch.empty((M, (K + 15) // 16 * 16), dtype=torch.int8, device=device)[:, :K]


def _output(out, out_dtype, M: int, N: int, device):
    torch = _torch()
    if out is None:
        _dtype_code(out_dtype)
        return torch.empty((M, N), dtype=out_dtype, device=device)
    _matrix("out", out, out_dtype)
    _dtype_code(out_dtype)
    if out.device != device or out.shape != (M, N):
        raise ValueError(f"out must be a [{M}, {N}] tensor on {device}")
    return out


def quantize_rows(x) -> Tuple["object", "object"]:
    """(integers [M, K] int8, scales [M] fp32) of ``x`` [M, K], a CUDA fp32,
    bf16 or fp16 tensor; the integers' rows lie a multiple of 16 bytes apart,
    as ``int8_matmul`` reads them."""
    torch = _torch()
    _matrix("x", x)
    code = _dtype_code(x.dtype)
    M, K = x.shape
    _check_inner(K)
    q = _empty_rows(M, K, x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    rc = launch(x.device, _lib.lib().ms_quantize_rows, x.data_ptr(), code, M, K, _pitch(x), q.data_ptr(), q.stride(0),
                scale.data_ptr())
    _lib.check(rc, "ms_quantize_rows")
    return q, scale


def _check_rows(name: str, t) -> int:
    pitch = t.stride(0) if t.shape[0] > 1 else (_pitch(t) + 15) // 16 * 16
    if pitch % 16 or t.data_ptr() % 16:
        raise ValueError(f"{name}'s rows must start 16-byte aligned (quantize_rows and Int8Linear lay them out so)")
    return pitch


def int8_matmul(xq, x_scale, wq, w_scale, *, bias=None, out_dtype=None, out=None):
    """``(xq @ wq.T) * x_scale[:, None] * w_scale + bias`` of integer matrices
    ``xq`` [M, K] and ``wq`` [N, K] with fp32 scales, rows 16-byte aligned;
    ``xq`` within [-127, 127], as ``quantize_rows`` makes it.
    Returns [M, N] in ``out_dtype`` (default: out's type, or fp32)."""
    torch = _torch()
    _matrix("xq", xq, torch.int8)
    _matrix("wq", wq, torch.int8)
    M, K = xq.shape
    N = wq.shape[0]
    if wq.shape[1] != K or wq.device != xq.device or N < 1:
        raise ValueError(f"wq must be a [N, {K}] tensor on {xq.device}")
    _check_inner(K)
    _vector("x_scale", x_scale, M, xq.device)
    _vector("w_scale", w_scale, N, xq.device)
    if bias is not None:
        _vector("bias", bias, N, xq.device)
    ldx, ldw = _check_rows("xq", xq), _check_rows("wq", wq)
    if out_dtype is None:
        out_dtype = torch.float32 if out is None else out.dtype
    out = _output(out, out_dtype, M, N, xq.device)
    rc = launch(xq.device, _lib.lib().ms_int8_matmul, xq.data_ptr(), ldx, x_scale.data_ptr(), M, wq.data_ptr(), ldw,
                w_scale.data_ptr(), N, K, None if bias is None else bias.data_ptr(), out.data_ptr(),
                _dtype_code(out_dtype), _pitch(out))
    _lib.check(rc, "ms_int8_matmul")
    return out


class Int8Linear:
    """A linear layer with int8 weights [N, K], one fp32 scale a channel.

    The weights are laid out once (rows a multiple of 16 bytes apart); a call
    quantises its tokens and multiplies, two launches of which the second's
    weight loads start under the first.
    """

    def __init__(self, weight, scale, bias=None) -> None:
        torch = _torch()
        _matrix("weight", weight, torch.int8)
        N, K = weight.shape
        if N < 1:
            raise ValueError("weight has no channels")
        _check_inner(K)
        self.scale = _vector("scale", scale, N, weight.device)
        self.bias = None if bias is None else _vector("bias", bias, N, weight.device)
        if weight.data_ptr() % 16 or _pitch(weight) % 16:
            rows = _empty_rows(N, K, weight.device)
            rows.copy_(weight)
            weight = rows
        self.weight = weight

    @classmethod
    def from_float(cls, weight, bias=None) -> "Int8Linear":
        """Quantise a float [N, K] weight, a scale for each channel."""
        q, scale = quantize_rows(weight)
        return cls(q, scale, bias)

    def __call__(self, x, *, out_dtype=None, out=None):
        """[M, N] of ``x`` [M, K] (fp32, bf16 or fp16) in ``out_dtype``
        (default: out's type, or fp32 as the sampler's logits)."""
        entry = _lib.binding()
        try:
            return entry.int8_linear(x, self.weight, self.scale, self.bias, out_dtype, out)
        except entry.CallError as e:
            _lib.check(e.args[0], "ms_int8_linear")
            raise
