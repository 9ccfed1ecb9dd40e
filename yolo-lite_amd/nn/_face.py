"""What the Python faces of the direct C entry points (``nn/mx4.py``, ``nn/block_attention.py``) share."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib


def on_gpu(what: str, *tensors: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError(f"{what} runs on the GPU only (HIP kernel, no CPU fallback)")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} has no backward pass: detach its inputs or call it under torch.no_grad()")
        if dev is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on different devices ({dev} and {t.device})")
        dev = t.device
    return dev


def call(dev: torch.device, fn, what: str, *args) -> None:
    """fn(*args, stream) with ``dev`` as the current device, on its current stream."""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        _lib.check(rc, what)
