"""Block-sparse attention: every query reads the key blocks that a cheap score selects for it.

The network's dense attention (``YL_OP_ATTENTION``) reads all pairs of tokens of a map; on a long map most of them say little.
``block_select`` scores each block of keys by its mean key, ``block_attention`` reads the blocks that were picked:

    picked = block_select(q, k, block=64, topk=8, mask=mask)             # (batch, kv heads, nq, topk) int32
    out = block_attention(q, k, v, picked, block=64, mask=mask)          # (batch, nq, heads, dv)

q (batch, nq, heads, dk), k (batch, nk, kv heads, dk), v (batch, nk, kv heads, dv) in bf16 or fp16; heads a multiple of kv heads;
mask (batch, nk), true where a key may be read.  Everything runs on the GPU through ``yl_block_*`` (no CPU fallback), on the
current stream of the tensors' device; inference only, no autograd.
"""
from __future__ import annotations

from ctypes import byref
from typing import Optional

import torch

from .. import _lib
from ._face import call, on_gpu

_TYPES = {torch.bfloat16: _lib.YL_BF16, torch.float16: _lib.YL_F16}


def _heads(t: torch.Tensor):
    """A tensor (batch, tokens, heads, width) the kernels can read in place, copied only where it is not one; and its strides."""
    if t.data_ptr() % 16 or (t.stride(3) != 1 and t.shape[3] > 1) or any(s % 8 for s in t.stride()[:3]):
        t = t.clone(memory_format=torch.contiguous_format)
    return t, _lib.Heads(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _check(what: str, q: torch.Tensor, k: torch.Tensor, mask: Optional[torch.Tensor]):
    if q.dtype not in _TYPES or k.dtype != q.dtype:
        raise TypeError(f"{what}: q and k are both bf16 or both fp16, got {q.dtype} and {k.dtype}")
    if q.dim() != 4 or k.dim() != 4 or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{what}: q (batch, nq, heads, dk) and k (batch, nk, kv heads, dk) are needed, got {tuple(q.shape)} and {tuple(k.shape)}")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"{what}: {q.shape[2]} query heads for {k.shape[2]} kv heads")
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8) or mask.shape != (k.shape[0], k.shape[1]):
        raise ValueError(f"{what}: a mask is (batch, nk) in bool or uint8, got {tuple(mask.shape)} in {mask.dtype}")
    if mask.shape[1] > 1 and mask.stride(1) != 1 or mask.shape[0] > 1 and mask.stride(0) < mask.shape[1]:
        mask = mask.contiguous()
    return mask


def _workspace(what: str, nbytes: int, like: torch.Tensor):
    if nbytes < 0:
        _lib.check(-3, what)
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def block_select(q: torch.Tensor, k: torch.Tensor, block: int = 64, topk: int = 8, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """For each query and kv head the ``topk`` blocks of ``block`` (32, 64 or 128) keys with the largest score, as int32
    (batch, kv heads, nq, topk): ascending block indices, -1 behind the last.  Score: (q summed over the kv head's query heads) .
    (mean of the block's readable keys), in 64 bits; ties go to the lower index; a block without a readable key is never picked."""
    dev = on_gpu("block_select", q, k, mask)
    mask = _check("block_select", q, k, mask)
    batch, nq, heads, dk = q.shape
    nk, kv = k.shape[1], k.shape[2]
    L = _lib.lib()
    nbytes = L.yl_block_select_workspace_bytes(batch, nq, nk, heads, kv, dk, block)
    work = _workspace("block_select", nbytes, q)
    q, qh = _heads(q)
    k, kh = _heads(k)
    picked = q.new_empty((batch, kv, nq, topk), dtype=torch.int32)
    call(dev, L.yl_block_select, "block_select", byref(qh), byref(kh), _TYPES[q.dtype], batch, nq, nk, heads, kv, dk, block, topk,
         mask.data_ptr() if mask is not None else None, mask.stride(0) if mask is not None else 0, picked.data_ptr(),
         work.data_ptr() if work is not None else None, nbytes)
    return picked


def block_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, picked: torch.Tensor, block: int = 64,
                    mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax over the readable keys of the picked blocks of ``scale`` q . k (default: dk ** -0.5), times v: (batch, nq, heads, dv).

    picked: int32 (batch, kv heads, nq, topk), as ``block_select`` gives it; entries that name no block are skipped and a block
    named twice counts once.  A query without a readable key gets zeros."""
    dev = on_gpu("block_attention", q, k, v, picked, mask)
    mask = _check("block_attention", q, k, mask)
    batch, nq, heads, dk = q.shape
    nk, kv = k.shape[1], k.shape[2]
    if v.dtype != q.dtype or v.dim() != 4 or v.shape[:3] != k.shape[:3]:
        raise ValueError(f"block_attention: v (batch, nk, kv heads, dv) in q's type is needed, got {tuple(v.shape)} in {v.dtype}")
    if picked.dtype != torch.int32 or picked.dim() != 4 or picked.shape[:3] != (batch, kv, nq):
        raise ValueError(f"block_attention: picked (batch, kv heads, nq, topk) in int32 is needed, got {tuple(picked.shape)} in {picked.dtype}")
    dv, topk = v.shape[3], picked.shape[3]
    L = _lib.lib()
    nbytes = L.yl_block_attention_workspace_bytes(_TYPES[q.dtype], batch, nq, nk, heads, kv, dk, dv, block, topk)
    work = _workspace("block_attention", nbytes, q)
    q, qh = _heads(q)
    k, kh = _heads(k)
    v, vh = _heads(v)
    picked = picked.contiguous()
    out = q.new_empty((batch, nq, heads, dv))
    oh = _lib.Heads(out.data_ptr(), out.stride(0), out.stride(1), out.stride(2))
    call(dev, L.yl_block_attention, "block_attention", byref(qh), byref(kh), byref(vh), _TYPES[q.dtype], batch, nq, nk, heads, kv, dk, dv,
         block, topk, picked.data_ptr(), mask.data_ptr() if mask is not None else None, mask.stride(0) if mask is not None else 0,
         dk ** -0.5 if scale is None else float(scale), byref(oh), work.data_ptr() if work is not None else None, nbytes)
    return out
