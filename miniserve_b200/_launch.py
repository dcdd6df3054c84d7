"""What every call of the decode-step operators does on the host besides its
own checks, kept short: a decode step makes dozens of them, and the kernels of
a small batch take a few microseconds."""
from __future__ import annotations

from .sampler import _torch


def launch(device, fn, *args) -> int:
    """``fn(*args, stream)`` with ``device`` current and its current stream."""
    torch = _torch()
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        return fn(*args, stream)
    with torch.cuda.device(device):
        return fn(*args, stream)


def refuse(name: str, t, shape, dtype, device, unit: bool = True) -> None:
    """Raise for a tensor that is not of this type, device and shape (None: any
    size), or not contiguous in its last dimension."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dim() != len(shape) or any(want is not None and got != want for got, want in zip(t.shape, shape)):
        want = ", ".join("any" if n is None else str(n) for n in shape)
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({want})")
    if unit and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
