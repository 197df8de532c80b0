"""8-bit activations with 4-bit weights without a GPU: the oracle of MXINT8, sizes, plans, refusals."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mxint8 as omi

E_SHAPE, E_ALIGN, E_FORMAT, E_WORKSPACE, E_NULL = -1, -2, -3, -5, -6


# ---------------------------------------------------------------- the oracle


def test_the_oracle_rounds_and_saturates():
    x = np.zeros((1, 64))
    x[0, :8] = [1.0, 1.5 / 64, 2.5 / 64, -0.5 / 64, 1.999, -1.999, 127.5 / 64, 0.49 / 64]
    x[0, 32] = 2.0 ** -140
    q, s = omi.quantize(x)
    assert list(q[0, :8]) == [64, 2, 2, 0, 127, -127, 127, 0]
    assert list(s[0]) == [127, 7] and q[0, 32] == 0
    assert omi.dequantize(q, s)[0, 0] == 1.0 and omi.dequantize(q, s)[0, 1] == 2 / 64
    x[0, 3] = np.inf
    q, s = omi.quantize(x)
    assert s[0, 0] == 255 and (q[0, :32] == 0).all() and np.isnan(omi.dequantize(q, s)[0, :32]).all()
    q, s = omi.quantize(np.full((1, 32), 2.0 ** 127))
    assert s[0, 0] == 253 and (q == 127).all()


def test_the_oracles_groups_can_be_read_back():
    """The 16 bytes of a group give every digit back by the places that the layout states."""
    rng = np.random.default_rng(0)
    for q in (rng.integers(-127, 128, 16), np.full(16, 127), np.full(16, -64), np.arange(-8, 8) * 15):
        word = int.from_bytes(omi.group_bytes(q, q < 0).tobytes(), "little")
        for i, v in enumerate(q):
            low = (word >> 6 * i) & 15
            high = (word >> (6 * i - 32) % 96) & 1
            high |= sum((((word >> 96) >> (6 * i + b) % 32) & 1) << b for b in (1, 2))
            assert 16 * high + low == abs(int(v)) and ((word >> (6 * i + 5)) & 1) == (v < 0)


# ---------------------------------------------------------------- sizes


@pytest.mark.parametrize("rows,cols", [(1, 32), (32, 256), (33, 288), (2048, 17408), (777, 1056)])
def test_packed_bytes(pkg, rows, cols):
    assert pkg.lib().qmlp_mxint8_bytes(rows, cols) == omi.packed_bytes(rows, cols)


def test_packed_bytes_refuses(pkg):
    for rows, cols in ((0, 32), (1, 16), (1, 0), (1, 33), (-1, 32), (1 << 21, 32), (1, 1 << 21)):
        assert pkg.lib().qmlp_mxint8_bytes(rows, cols) == 0


def test_workspaces_never_shrink_as_m_grows(pkg):
    lib = pkg.lib()
    Ms = list(range(1, 700)) + [1023, 1024, 2047, 2048, 2049, 65536]
    for N, K in ((5120, 17408), (17408, 5120), (100, 32), (1, 1056)):
        for x_type in (0, 1, 2, 4):
            sizes = [lib.qmlp_w4a8_workspace_bytes(M, N, K, x_type) for M in Ms]
            assert sizes[Ms.index(33)] > 0 and sizes == sorted(sizes)
            assert (sizes[Ms.index(32)] == 0) == (x_type == 4)
    for bad in ((0, 256, 256), (65537, 256, 256), (1, 0, 256), (1, 256, 48)):
        assert lib.qmlp_w4a8_workspace_bytes(*bad, 0) == 0
PLAN_SHAPES = []
