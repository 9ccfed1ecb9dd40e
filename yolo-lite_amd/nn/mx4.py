"""4-bit microscaled tensors (OCP microscaling, e2m1 elements, one e8m0 scale per 32 columns) and products with them.

The step below the e4m3 convs of ``nn/lower.py``: a pointwise conv is ``mx4_linear`` over pixels as rows.  Everything runs on the
GPU through ``yl_mx4_*`` (no CPU fallback), on the current stream of the tensors' device; inference only, no autograd.

    w = mx4_quantize(weight)                       # (n, k) once
    y = mx4_linear(x, w, bias=b, act=True)         # x (..., k) in bf16 / fp16 / fp32: quantised on the way
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from .. import _lib
from ._face import call as _call, on_gpu as _on_gpu

BLOCK = 32  # columns that share one scale
_TYPES = {torch.bfloat16: _lib.YL_BF16, torch.float32: _lib.YL_F32, torch.float16: _lib.YL_F16}


class Mx4Tensor(NamedTuple):
    """A matrix in MX4.  ``codes`` uint8 (..., ceil(cols / 32) * 16): two codes to a byte, the first in the low half;
    ``scales`` uint8 (..., ceil(cols / 32)): s stands for 2^(s - 127), 255 for NaN; ``cols``: columns of the matrix."""

    codes: torch.Tensor
    scales: torch.Tensor
    cols: int


def _rows(x: torch.Tensor) -> torch.Tensor:
    """(..., k) as (rows, k) with unit column stride; copied only where no such view exists."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    (rows, cols), (step, one) = x.shape, x.stride()
    if one != 1 and cols > 1 or rows > 1 and step < cols:
        x = x.contiguous()
    return x


def _dense(what: str, t: Mx4Tensor):
    """Codes and scales as dense 2-d arrays of matching shapes."""
    codes, scales, cols = t
    kb = (cols + BLOCK - 1) // BLOCK
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"{what}: codes and scales are uint8 tensors")
    cs, ss = codes.shape, scales.shape
    if cols < 1 or len(ss) == 0 or ss[-1] != kb or cs != (*ss[:-1], kb * 16):
        raise ValueError(f"{what}: codes {tuple(cs)} and scales {tuple(ss)} do not hold {cols} columns")
    if not codes.is_contiguous() or codes.data_ptr() & 15:
        codes = codes.clone(memory_format=torch.contiguous_format)
    return codes, scales if scales.is_contiguous() else scales.contiguous()


def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """(..., cols) in bf16, fp16 or fp32 -> ``Mx4Tensor``.  Round to nearest even, saturating; a block of 32 columns that holds an
    infinity or a NaN reads as NaN."""
    dev = _on_gpu("mx4_quantize", x)
    if x.dtype not in _TYPES:
        raise TypeError(f"mx4_quantize: bf16, fp16 or fp32 values, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"mx4_quantize: no columns in a tensor of shape {tuple(x.shape)}")
    lead, cols = x.shape[:-1], x.shape[-1]
    kb = (cols + BLOCK - 1) // BLOCK
    x = _rows(x)
    codes = x.new_empty((*lead, kb * 16), dtype=torch.uint8)
    scales = x.new_empty((*lead, kb), dtype=torch.uint8)
    _call(dev, _lib.lib().yl_mx4_quantize, "mx4_quantize", x.data_ptr(), _TYPES[x.dtype], x.shape[0], cols, max(x.stride(0), cols),
          codes.data_ptr(), scales.data_ptr())
    return Mx4Tensor(codes, scales, cols)


def mx4_dequantize(t: Mx4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values an ``Mx4Tensor`` stands for (exact in bf16 and fp32)."""
    dev = _on_gpu("mx4_dequantize", t.codes, t.scales)
    if dtype not in _TYPES:
        raise TypeError(f"mx4_dequantize: bf16, fp16 or fp32 values, got {dtype}")
    codes, scales = _dense("mx4_dequantize", t)
    y = codes.new_empty((*codes.shape[:-1], t.cols), dtype=dtype)
    _call(dev, _lib.lib().yl_mx4_dequantize, "mx4_dequantize", codes.data_ptr(), scales.data_ptr(), y.numel() // t.cols, t.cols,
          y.data_ptr(), _TYPES[dtype], t.cols)
    return y


def mx4_linear(x: Union[torch.Tensor, Mx4Tensor], w: Mx4Tensor, bias: Optional[torch.Tensor] = None, act: bool = False,
               res: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(x w^T + bias) + res`` with both operands in MX4 and fp32 accumulation.

    x: (..., k) values, quantised by the call, or an ``Mx4Tensor``; w: ``Mx4Tensor`` (n, k); bias: (n,) (used in fp32);
    act: SiLU; res: (..., n) in the result's type, added after the activation.  dtype: the result's type (default: x's; bf16 for
    an ``Mx4Tensor``)."""
    packed = isinstance(x, Mx4Tensor)
    xt = x.codes if packed else x
    dev = _on_gpu("mx4_linear", xt, w.codes, w.scales, bias, res)
    if w.codes.dim() != 2:
        raise ValueError(f"mx4_linear: the weight is a matrix (n, k), got codes of shape {tuple(w.codes.shape)}")
    wc, ws = _dense("mx4_linear", w)
    n, k = wc.shape[0], w.cols
    if n == 0:
        raise ValueError("mx4_linear: the weight has no rows")
    if packed:
        _on_gpu("mx4_linear", xt, x.scales)
        xt, xs = _dense("mx4_linear", x)
        cols, in_type, stride = x.cols, _lib.YL_MX4, x.cols
    else:
        if xt.dtype not in _TYPES:
            raise TypeError(f"mx4_linear: bf16, fp16 or fp32 activations, got {xt.dtype}")
        if xt.dim() == 0:
            raise ValueError("mx4_linear: activations (..., k) are needed")
        cols, in_type, xs = xt.shape[-1], _TYPES[xt.dtype], None
    if cols != k:
        raise ValueError(f"mx4_linear: activations of {cols} columns and a weight of {k}")
    dtype = dtype or (torch.bfloat16 if packed else xt.dtype)
    if dtype not in _TYPES:
        raise TypeError(f"mx4_linear: bf16, fp16 or fp32 results, got {dtype}")
    lead = xt.shape[:-1]
    rows = 1
    for d in lead:
        rows *= d
    if not packed:
        xt = _rows(xt)
        stride = max(xt.stride(0), k)
    if bias is not None:
        if bias.shape != (n,):
            raise ValueError(f"mx4_linear: a bias of shape {tuple(bias.shape)} for {n} output columns")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.float().contiguous()
    if res is not None:
        if res.shape != (*lead, n) or res.dtype != dtype:
            raise ValueError(f"mx4_linear: a residual {tuple(res.shape)} in {res.dtype} for a result {(*lead, n)} in {dtype}")
        res = _rows(res)
    y = wc.new_empty((*lead, n), dtype=dtype)
    L = _lib.lib()
    nbytes = L.yl_mx4_linear_workspace_bytes(in_type, rows, n, k)
    if nbytes < 0:
        _lib.check(-3, "mx4_linear")
    work = wc.new_empty(nbytes) if nbytes else None
    _call(dev, L.yl_mx4_linear, "mx4_linear", xt.data_ptr(), xs.data_ptr() if xs is not None else None, in_type, rows, stride,
          wc.data_ptr(), ws.data_ptr(), n, k, bias.data_ptr() if bias is not None else None, int(bool(act)),
          res.data_ptr() if res is not None else None, max(res.stride(0), n) if res is not None else 0, y.data_ptr(), _TYPES[dtype], n,
          work.data_ptr() if work is not None else None, nbytes)
    return y
