"""A call of the library on a tensor's device and its current stream."""
from __future__ import annotations

from .sampler import _torch


def launch(device, fn, *args) -> int:
    """``fn(*args, stream)`` with ``device`` current and its current stream."""
    torch = _torch()
    with torch.cuda.device(device):
        return fn(*args, torch.cuda.current_stream(device).cuda_stream)
