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

import struct
from typing import Optional

import torch

from .. import _lib
from ._face import call, on_gpu

_TYPES = {torch.bfloat16: _lib.YL_BF16, torch.float16: _lib.YL_F16}


_pack = struct.Struct("Pqqq").pack  # a yl_heads


def _heads(t: torch.Tensor):
    """A tensor (batch, tokens, heads, width) the kernels can read in place, copied only where it is not one; and its yl_heads."""
    at, (b, n, h, c) = t.data_ptr(), t.stride()
    if at & 15 or (b | n | h) & 7 or (c != 1 and t.shape[3] > 1):
        t = t.clone(memory_format=torch.contiguous_format)
        at, (b, n, h, c) = t.data_ptr(), t.stride()
    return t, _pack(at, b, n, h)


def _check(what: str, q: torch.Tensor, k: torch.Tensor, mask: Optional[torch.Tensor], block: int, topk: int):
    """-> the sizes batch, nq, heads, dk, nk, kv heads; and the mask as rows of bytes, its address and row stride."""
    if q.dtype not in _TYPES or k.dtype != q.dtype:
        raise TypeError(f"{what}: q and k are both bf16 or both fp16, got {q.dtype} and {k.dtype}")
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[0] != ks[0] or qs[3] != ks[3]:
        raise ValueError(f"{what}: q (batch, nq, heads, dk) and k (batch, nk, kv heads, dk) are needed, got {tuple(qs)} and {tuple(ks)}")
    batch, nq, heads, dk = qs
    nk, kv = ks[1], ks[2]
    if (batch | nq | heads | nk | block | topk) >> 31:  # (the C calls take 32-bit sizes; a larger one would wrap)
        raise NotImplementedError(f"{what}: sizes from 0 to {2 ** 31 - 1}, got q {tuple(qs)}, k {tuple(ks)}, block {block}, topk {topk}")
    if kv == 0 or heads == 0 or heads % kv:
        raise ValueError(f"{what}: {heads} query heads for {kv} kv heads")
    at = row = None
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.shape != (batch, nk):
            raise ValueError(f"{what}: a mask is (batch, nk) in bool or uint8, got {tuple(mask.shape)} in {mask.dtype}")
        row, one = mask.stride()
        if nk > 1 and one != 1 or batch > 1 and row < nk:
            mask = mask.contiguous()
            row = nk
        at = mask.data_ptr()
    return qs, nk, kv, mask, at, row or 0


def _workspace(what: str, nbytes: int, like: torch.Tensor):
    if nbytes < 0:
        _lib.check(-3, what)
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def block_select(q: torch.Tensor, k: torch.Tensor, block: int = 64, topk: int = 8, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """For each query and kv head the ``topk`` blocks of ``block`` (32, 64 or 128) keys with the largest score, as int32
    (batch, kv heads, nq, topk): ascending block indices, -1 behind the last.  Score: (q summed over the kv head's query heads) .
    (mean of the block's readable keys), in 64 bits; ties go to the lower index, a NaN score ranks with -inf; a block without a readable
    key is never picked."""
    dev = on_gpu("block_select", q, k, mask)
    (batch, nq, heads, dk), nk, kv, mask, mask_at, mask_row = _check("block_select", q, k, mask, block, topk)
    L = _lib.lib()
    nbytes = L.yl_block_select_workspace_bytes(batch, nq, nk, heads, kv, dk, block)
    work = _workspace("block_select", nbytes, q)
    q, qh = _heads(q)
    k, kh = _heads(k)
    picked = q.new_empty((batch, kv, nq, topk), dtype=torch.int32)
    call(dev, L.yl_block_select, "block_select", qh, kh, _TYPES[q.dtype], batch, nq, nk, heads, kv, dk, block, topk, mask_at, mask_row,
         picked.data_ptr(), work.data_ptr() if work is not None else None, nbytes)
    return picked


def block_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, picked: torch.Tensor, block: int = 64,
                    mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax over the readable keys of the picked blocks of ``scale`` q . k (default: dk ** -0.5), times v: (batch, nq, heads, dv).

    picked: int32 (batch, kv heads, nq, topk), as ``block_select`` gives it; entries that name no block are skipped and a block
    named twice counts once.  A query without a readable key gets zeros.  Sums are fp32; weights are rounded to the tensors' type before
    they multiply v, and for bf16 a block's result may be rounded to fp16 (2^-11 of its sum of weights times |v|)."""
    dev = on_gpu("block_attention", q, k, v, picked, mask)
    vs, ps = v.shape, picked.shape
    topk = ps[3] if len(ps) == 4 else 0
    (batch, nq, heads, dk), nk, kv, mask, mask_at, mask_row = _check("block_attention", q, k, mask, block, topk)
    if v.dtype != q.dtype or len(vs) != 4 or vs[:3] != (batch, nk, kv):
        raise ValueError(f"block_attention: v (batch, nk, kv heads, dv) in q's type is needed, got {tuple(vs)} in {v.dtype}")
    if picked.dtype != torch.int32 or len(ps) != 4 or ps[:3] != (batch, kv, nq):
        raise ValueError(f"block_attention: picked (batch, kv heads, nq, topk) in int32 is needed, got {tuple(ps)} in {picked.dtype}")
    dv = vs[3]
    L = _lib.lib()
    nbytes = L.yl_block_attention_workspace_bytes(_TYPES[q.dtype], batch, nq, nk, heads, kv, dk, dv, block, topk)
    work = _workspace("block_attention", nbytes, q)
    q, qh = _heads(q)
    k, kh = _heads(k)
    v, vh = _heads(v)
    picked = picked.contiguous()
    out = q.new_empty((batch, nq, heads, dv))
    oh = _pack(out.data_ptr(), nq * heads * dv, heads * dv, dv)
    call(dev, L.yl_block_attention, "block_attention", qh, kh, vh, _TYPES[q.dtype], batch, nq, nk, heads, kv, dk, dv, block, topk,
         picked.data_ptr(), mask_at, mask_row, dk ** -0.5 if scale is None else float(scale), oh,
         work.data_ptr() if work is not None else None, nbytes)
    return out
