"""MX4 (e2m1 elements, e8m0 scales, blocks of 32) restated in numpy on 64-bit floats, from the definition alone."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(x: np.ndarray) -> np.ndarray:
    """(rows, cols) -> (rows, blocks, 32) in 64 bits, zeros behind the last column."""
    rows, cols = x.shape
    kb = -(-cols // 32)
    v = np.zeros((rows, kb * 32))
    v[:, :cols] = x
    return v.reshape(rows, kb, 32)


def quantize(x: np.ndarray):
    """-> codes 0..15 (rows, blocks, 32) and scale bytes (rows, blocks)."""
    v = blocks(x.astype(np.float64))
    finite = np.isfinite(v).all(-1)
    amax = np.where(finite, np.abs(np.where(np.isfinite(v), v, 0)).max(-1), 1.0)
    _, e = np.frexp(amax)
    byte = np.where(amax > 0, np.maximum(e - 1 - 2, -127) + 127, 0)
    a = np.minimum(np.abs(np.where(finite[..., None], v, 0.0)) / np.ldexp(1.0, byte - 127)[..., None], 6.0)
    d = np.abs(a[..., None] - LEVELS)
    near = d.min(-1, keepdims=True) == d
    # a tie goes to the even code
    code = np.argmax(near * (1 + (np.arange(8) % 2 == 0)), -1)
    code = code + 8 * np.signbit(v)
    return code.astype(np.int64), np.where(finite, byte, 255).astype(np.int64)


def pack(code: np.ndarray) -> np.ndarray:
    c = code.reshape(code.shape[0], -1)
    return (c[:, 0::2] | c[:, 1::2] << 4).astype(np.uint8)


def unpack(codes: np.ndarray) -> np.ndarray:
    c = np.stack((codes & 15, codes >> 4), -1).astype(np.int64)
    return c.reshape(codes.shape[0], -1, 32)


def values(code: np.ndarray, byte: np.ndarray, cols: int) -> np.ndarray:
    v = LEVELS[code & 7] * np.where(code > 7, -1.0, 1.0) * np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))[..., None]
    return v.reshape(code.shape[0], -1)[:, :cols]


def rounded(x: np.ndarray) -> np.ndarray:
    """What quantising x and reading it back gives."""
    return values(*quantize(x), x.shape[1])
