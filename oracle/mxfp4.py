"""MXFP4 (OCP microscaled 4-bit floating point) oracle in numpy: the definition of the format, in 64
bits, and the library's packed layout.  Plain and slow; nothing in the package imports it.

A block is 32 consecutive values of a row.  Its scale is 2^(s - 127) with s a byte (255: not a number);
its elements are e2m1: the code's low three bits index VALUES, bit 3 is the sign.
"""
import numpy as np

BLOCK = 32
VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
UNIT_ROWS, UNIT_K, UNIT_BYTES = 32, 256, 4352
TRAILER_BYTES, TRAILER_MAGIC = 256, 0x514D4C50


def nearest_codes(v):
    """e2m1 codes of float64 values: the nearest of +-VALUES, a tie to the even index, beyond 6 to 6."""
    a = np.minimum(np.abs(v), 6.0)
    d = np.abs(a[..., None] - VALUES)
    best = d.min(axis=-1, keepdims=True)
    tied = d == best
    even = np.where(tied, np.arange(8) % 2, 2).argmin(axis=-1)  # an even index if one is among the nearest
    return (even + 8 * np.signbit(v)).astype(np.uint8)


def quantize(x):
    """float array [rows, cols] -> codes [rows, cols] (one to a byte), scales [rows, cols / 32]."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    b = x.reshape(rows, cols // BLOCK, BLOCK)
    top = np.abs(b).max(axis=2)
    finite = np.isfinite(b).all(axis=2)
    _, e = np.frexp(np.where(finite, top, 1.0))
    e = np.where(top > 0, e - 1, -10000)
    e = np.maximum(e, -124) - 2
    codes = nearest_codes(np.ldexp(np.where(finite[..., None], b, 0.0), -e[..., None]))
    codes = np.where(finite[..., None], codes, 0).astype(np.uint8)
    scales = np.where(finite, e + 127, 255).astype(np.uint8)
    return codes.reshape(rows, cols), scales


def dequantize(codes, scales):
    """codes [rows, cols] (one to a byte), scales -> float64 values (NaN where the scale is 255)."""
    v = np.concatenate([VALUES, -VALUES])[codes].reshape(codes.shape[0], -1, BLOCK)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(codes.shape)


def join(codes):
    """Two codes to a byte, the even column in the low half."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def split(joined):
    out = np.empty((joined.shape[0], 2 * joined.shape[1]), dtype=np.uint8)
    out[:, 0::2], out[:, 1::2] = joined & 15, joined >> 4
    return out


def packed_bytes(rows, cols):
    return -(-rows // UNIT_ROWS) * -(-cols // UNIT_K) * UNIT_BYTES + TRAILER_BYTES


def pack(codes, scales):
    """The packed layout's bytes: units of 32 rows x 256 K, then the trailer."""
    rows, cols = codes.shape
    nsb = -(-cols // UNIT_K)
    out = np.zeros((-(-rows // UNIT_ROWS), nsb, UNIT_BYTES), dtype=np.uint8)
    out[:, :, 4096:] = 1
    j = join(codes)
    for r in range(rows):
        for g in range(cols // BLOCK):
            unit = out[r // UNIT_ROWS, g // 8]
            kb, row = g % 8, r % UNIT_ROWS
            at = (kb * UNIT_ROWS + row) * 16
            unit[at:at + 16] = j[r, 16 * g:16 * g + 16]
            unit[4096 + 4 * (row + UNIT_ROWS * (kb % 2)) + kb // 2] = scales[r, g]
    trailer = np.zeros(TRAILER_BYTES // 4, dtype=np.uint32)
    trailer[3] = TRAILER_MAGIC
    trailer[4] = int((scales == 255).sum())
    return np.concatenate([out.reshape(-1), trailer.view(np.uint8)])


def linear(a, b):
    """(a b^T, |a| |b|^T) in float64 for dequantised operands: the product and what bounds its rounding."""
    with np.errstate(invalid="ignore"):
        return a @ b.T, np.abs(a) @ np.abs(b).T
