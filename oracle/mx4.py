"""The 4-bit KV cache format in numpy, from its definition.

Rows of D elements in blocks of 32: a scale byte b per block, standing for
2^(b - 127), and a 4-bit code per element, sign and magnitude
0 .5 1 1.5 2 3 4 6. The 8-element chunk c of a row is the 4-byte unit
(c % 4) * (D / 32) + c / 4; its element i is in bits 4 i .. 4 i + 3 of the unit.
No counterpart in the reference, whose backend refuses a quantised cache
(fxpr_vllm/attention_backend.py:40-277).
"""

from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# scale bytes a writer gives the type; a reader takes a larger one as the last
BYTES = {"f16": (104, 140), "bf16": (2, 252), "f32": (2, 252)}


def _place(d: int) -> tuple[np.ndarray, np.ndarray]:
    """(byte, shift) of each of the d elements of a row."""
    e = np.arange(d)
    chunk, i = e // 8, e % 8
    return 4 * ((chunk % 4) * (d // 32) + chunk // 4) + i // 2, 4 * (i % 2)


def pack(codes: np.ndarray) -> np.ndarray:
    """4-bit codes [..., D] -> bytes [..., D / 2]."""
    d = codes.shape[-1]
    byte, shift = _place(d)
    out = np.zeros(codes.shape[:-1] + (d // 2,), np.uint8)
    for e in range(d):
        out[..., byte[e]] |= (codes[..., e] << shift[e]).astype(np.uint8)
    return out


def unpack(data: np.ndarray) -> np.ndarray:
    """Bytes [..., D / 2] -> 4-bit codes [..., D]."""
    byte, shift = _place(2 * data.shape[-1])
    return (data[..., byte] >> shift.astype(np.uint8)) & 15


def quantise(x: np.ndarray, dtype: str) -> tuple[np.ndarray, np.ndarray]:
    """Values [..., D] (float64 holding `dtype` values) -> (codes [..., D], scale bytes [..., D / 32])."""
    lo, hi = BYTES[dtype]
    blocks = np.where(np.isnan(x), 0.0, x).reshape(x.shape[:-1] + (-1, 32))
    amax = np.minimum(np.abs(blocks).max(-1), 2.0 ** 129)  # (an infinity: above every limit)
    _, e = np.frexp(np.where(amax > 0, amax, 2.0 ** -200))
    p = e - 1  # amax in [2^p, 2^(p + 1))
    p = np.where(amax > 1.75 * 2.0 ** p.astype(np.float64), p + 1, p) - 2
    b = np.clip(p + 127, lo, hi)
    y = np.abs(blocks) / 2.0 ** (b[..., None] - 127.0)
    dist = np.abs(np.minimum(y, 6.0)[..., None] - MAGNITUDES)
    # the nearest magnitude (the distances are exact where two are equal); of two
    # equally near ones the even code
    near = dist == dist.min(-1, keepdims=True)
    code = (near * (2 - np.arange(8) % 2)).argmax(-1) + 8 * np.signbit(blocks)
    return code.reshape(x.shape).astype(np.uint8), b.astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray, dtype: str) -> np.ndarray:
    """float64 values of 4-bit codes [..., D] and scale bytes [..., D / 32]."""
    b = np.minimum(scales.astype(np.int64), BYTES[dtype][1])
    mag = MAGNITUDES[codes & 7] * np.repeat(2.0 ** (b - 127.0), 32, axis=-1)
    return np.where(codes & 8, -mag, mag)
