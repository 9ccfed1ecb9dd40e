"""What the Python faces of the direct C entry points (``nn/mx4.py``, ``nn/block_attention.py``) share.  A small call is bound by the
host (an allocation and a launch are 2-4 us each), so the checks are a few attribute reads and the message is made when one fails."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _lib


def on_gpu(what: str, *tensors: Optional[torch.Tensor]) -> int:
    """The index of the one GPU all of the tensors are on; raises for tensors elsewhere, on two GPUs, or that want a gradient or carry a
    tangent."""
    at = -1
    tangents = forward_ad._current_level >= 0  # (inside forward_ad.dual_level())
    for t in tensors:
        if t is None:
            continue
        d = t.get_device()
        if d < 0 or (at >= 0 and d != at) or t.requires_grad or tangents:
            _refuse(what, at, t)
        at = d
    return at


def _refuse(what: str, at: int, t: torch.Tensor) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} runs on the GPU only (HIP kernel, no CPU fallback)")
    if at >= 0 and t.device.index != at:
        raise ValueError(f"{what}: tensors on different devices (cuda:{at} and {t.device})")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:  # (no_grad does not stop forward mode)
        raise RuntimeError(f"{what} has no derivative: take the primal of its inputs (torch.autograd.forward_ad.unpack_dual)")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no backward pass: detach its inputs or call it under torch.no_grad()")


def call(dev: int, fn, what: str, *args) -> None:
    """fn(*args, stream) with ``dev`` as the current device, on its current stream."""
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, what)
