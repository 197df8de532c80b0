"""MXINT8 (OCP microscaled 8-bit integers) oracle in numpy: the definition of the format, in 64 bits, and the
library's packed layout.  Plain and slow; nothing in the package imports it.

A block is 32 consecutive values of a row.  Its scale byte is s = E + 127 with E the binade of its largest
magnitude, kept in [-120, 126] (255: not a number); its elements are integers q in -127..127 that stand for
q 2^(E - 6).
"""
import numpy as np

BLOCK = 32
UNIT_ROWS, UNIT_K, UNIT_BYTES, PLANE_BYTES = 32, 256, 8448, 4096


def quantize(x):
    """float array [rows, cols] -> integers [rows, cols], scale bytes [rows, cols / 32]."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    b = x.reshape(rows, cols // BLOCK, BLOCK)
    finite = np.isfinite(b).all(axis=2)
    top = np.abs(np.where(finite[..., None], b, 0.0)).max(axis=2)
    e = np.where(top > 0, np.frexp(top)[1] - 1, -10000).clip(-120, 126)
    q = np.rint(np.ldexp(np.where(finite[..., None], b, 0.0), 6 - e[..., None])).clip(-127, 127)
    return q.astype(np.int8).reshape(rows, cols), np.where(finite, e + 127, 255).astype(np.uint8)


def dequantize(q, scales):
    """float64 values (NaN where the scale is 255)."""
    v = q.astype(np.float64).reshape(q.shape[0], -1, BLOCK)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 133))
    return (v * s[..., None]).reshape(q.shape)


def packed_bytes(rows, cols):
    return -(-rows // UNIT_ROWS) * -(-cols // UNIT_K) * UNIT_BYTES


def group_bytes(q, negative):
    """16 integers and the signs of what they were rounded from (zeros keep theirs) -> 16 bytes: 96 bits of 6-bit
    fields (sign, a bit of another digit, the low digit), then the two high bits of every high digit at their places
    modulo 32."""
    low = high = 0
    for i, v in enumerate(int(a) for a in q):
        low |= ((abs(v) & 15) | (32 if negative[i] else 0)) << 6 * i
        high |= (abs(v) >> 4) << 6 * i
    last = 0
    for i in range(16):
        # the low bit of field i's high digit, bit 6 i, is kept 32 bits before that, around the 96
        low |= ((high >> 6 * i) & 1) << (6 * i - 32) % 96
        for bit in (6 * i + 1, 6 * i + 2):
            last |= ((high >> bit) & 1) << bit % 32
    return np.frombuffer((low | last << 96).to_bytes(16, "little"), dtype=np.uint8)


def packed_rows(q, scales, negative):
    """{(offset): bytes} of what a packed matrix of these rows holds, padding up to the K unit's end included."""
    rows, cols = q.shape
    nsb = -(-cols // UNIT_K)
    for r in range(rows):
        for kb in range(nsb * 8):
            signs = negative[r, kb * BLOCK:(kb + 1) * BLOCK] & (scales[r, min(kb, cols // BLOCK - 1)] != 255)
            unit = ((r // UNIT_ROWS) * nsb + kb // 8) * UNIT_BYTES
            row, b = r % UNIT_ROWS, kb % 8
            inside = kb * BLOCK < cols
            block = q[r, kb * BLOCK:(kb + 1) * BLOCK] if inside else np.zeros(BLOCK, np.int8)
            signs = signs if inside else np.zeros(BLOCK, bool)
            for g in range(2):
                at = unit + g * PLANE_BYTES + (b // 2) * 1024 + (row + UNIT_ROWS * (b % 2)) * 16
                yield at, group_bytes(block[16 * g:16 * g + 16], signs[16 * g:16 * g + 16])
            s = int(scales[r, kb]) if inside else 7
            yield (unit + 2 * PLANE_BYTES + 4 * (row + UNIT_ROWS * (b % 2)) + b // 2,
                   np.array([s if s == 255 else s - 3], dtype=np.uint8))
