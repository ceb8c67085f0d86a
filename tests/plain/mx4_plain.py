"""Microscaled 4-bit floating point from its definition, in 64 bits, on the CPU."""

import numpy as np

BLOCK = 32
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """``x`` float64 [rows, columns] -> (codes uint8 [rows, blocks, 32], scale bytes uint8 [rows, blocks])."""
    x = np.asarray(x, dtype=np.float64)
    rows, columns = x.shape
    blocks = -(-columns // BLOCK)
    v = np.zeros((rows, blocks * BLOCK))
    v[:, :columns] = x
    v = v.reshape(rows, blocks, BLOCK)
    top = np.abs(v).max(axis=2)
    finite = np.isfinite(v).all(axis=2)
    _, e = np.frexp(np.where(finite, top, 1.0))         # top = m 2^e, 1/2 <= m < 1: floor(log2 top) = e - 1
    exponent = np.where((top > 0) | ~finite, np.clip(e - 3, -127, 127), -127)
    size = np.abs(np.where(finite[..., None], v, 0.0)) * np.exp2(-exponent.astype(np.float64))[..., None]
    distance = np.abs(size[..., None] - MAGNITUDES)
    nearest = distance == distance.min(axis=-1, keepdims=True)
    first = nearest.argmax(axis=-1)
    second = 7 - nearest[..., ::-1].argmax(axis=-1)
    code = np.where(first % 2 == 0, first, second)      # two candidates: neighbours, one of them even
    code = code | (np.signbit(v).astype(np.int64) << 3)
    code = np.where(finite[..., None], code, 0)
    scale = np.where(finite, exponent + 127, 255)
    return code.astype(np.uint8), scale.astype(np.uint8)


def values(codes, scales, columns):
    """What codes [rows, blocks, 32] and scale bytes stand for, float64 [rows, columns]."""
    v = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(codes.shape[0], -1)[:, :columns]


def stored(codes, columns):
    """Codes [rows, blocks, 32] as a file holds them: two a byte, the first in the low half, [rows, ceil(columns / 2)]."""
    flat = codes.reshape(codes.shape[0], -1)[:, :columns]
    if columns % 2:
        flat = np.pad(flat, ((0, 0), (0, 1)))
    return (flat[:, 0::2] | flat[:, 1::2] << 4).astype(np.uint8)

