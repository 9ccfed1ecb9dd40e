"""Block-sparse attention restated in numpy on 64-bit floats, query by query, from the definition alone."""
import numpy as np


def readable(nk, mask_row):
    return np.ones(nk, bool) if mask_row is None else np.asarray(mask_row, bool)


def select(q, k, block, topk, mask=None):
    """q (b, nq, heads, dk), k (b, nk, kv, dk) -> (b, kv, nq, topk)."""
    b, nq, heads, dk = q.shape
    nk, kv = k.shape[1:3]
    nb = -(-nk // block)
    out = np.full((b, kv, nq, topk), -1, np.int64)
    for i in range(b):
        ok = readable(nk, None if mask is None else mask[i])
        can = np.array([ok[j * block: (j + 1) * block].any() for j in range(nb)], bool)
        for h in range(kv):
            mean = np.zeros((nb, dk))
            for j in range(nb):
                if can[j]:
                    mean[j] = k[i, j * block: (j + 1) * block, h][ok[j * block: (j + 1) * block]].mean(0)
            qq = q[i, :, h * heads // kv: (h + 1) * heads // kv].sum(1)
            with np.errstate(invalid="ignore"):
                score = qq @ mean.T
            score[np.isnan(score)] = -np.inf
            for t in range(nq):
                order = sorted((j for j in range(nb) if can[j]), key=lambda j: (-score[t, j], j))[:topk]
                out[i, h, t, : len(order)] = sorted(order)
    return out


def attend(q, k, v, picked, block, mask=None, scale=None):
    """-> out (b, nq, heads, dv), and per output the sum of softmax weights times |v| and of |q k| behind the largest score."""
    b, nq, heads, dk = q.shape
    nk, kv = k.shape[1:3]
    scale = dk ** -0.5 if scale is None else scale
    out = np.zeros((b, nq, heads, v.shape[3]))
    mass, work = np.zeros_like(out), np.zeros((b, nq, heads, 1))
    of = np.arange(nk) // block
    for i in range(b):
        ok = readable(nk, None if mask is None else mask[i])
        for h in range(heads):
            g = h * kv // heads
            for t in range(nq):
                see = ok & np.isin(of, picked[i, g, t])
                if not see.any():
                    continue
                z = scale * (k[i, see, g] @ q[i, t, h])
                p = np.exp(z - z.max())
                p /= p.sum()
                out[i, t, h] = p @ v[i, see, g]
                mass[i, t, h] = p @ np.abs(v[i, see, g])
                work[i, t, h] = abs(scale) * (np.abs(k[i, see, g]) @ np.abs(q[i, t, h])).max()
    return out, mass, work
