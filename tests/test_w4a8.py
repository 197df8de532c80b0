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
    # what 16 tokens of packed activations or one quantised token need nothing for
    assert lib.qmlp_w4a8_workspace_bytes(1, 5120, 17408, 0) == 0 < lib.qmlp_w4a8_workspace_bytes(2, 5120, 17408, 0)


# ---------------------------------------------------------------- plans

# (matrices, M, N, K): sizes whose plans take every kernel that the products launch, whole, with the K range in
# pieces and with pieces behind whole tiles, quantising inside (in four and eight waves) and in front; the GPU tests
# run them all.
PLAN_SHAPES = [(1, 17, 33, 32), (1, 17, 5092, 2688), (1, 22, 33, 1152), (1, 814, 487, 1632), (1, 1089, 35, 32),
               (1, 1042, 39, 1856), (1, 2320, 1584, 32), (1, 2222, 47, 29888), (1, 841, 9533, 1632), (1, 5, 33, 32),
               (1, 1, 33, 32), (1, 1, 8200, 96), (1, 16, 8225, 96), (1, 3, 100, 5120), (2, 17, 33, 32),
               (2, 17, 256, 1056), (2, 18, 35, 1088), (2, 1029, 256, 32), (2, 34, 256, 12480), (2, 136, 13824, 32),
               (2, 73, 2816, 10304), (2, 1508, 2816, 1824), (2, 5, 256, 96), (2, 1, 256, 96), (2, 1, 8448, 96),
               (2, 2372, 769, 32), (2, 1362, 3035, 2080)]


def _plan(pkg, nmat, M, N, K, cus=256):
    """(kernel, pieces, workgroups, KB of partial tiles, quantises inside, tiles that run whole)"""
    out = (ctypes.c_int * 5)()
    assert pkg.lib().qmlp_w4a8_plan(M, N, K, nmat, cus, out) == 0
    kind, ks, groups, kb, inside = out
    whole = 0
    if kind in (4, 5) and ks > 1:
        tiles = -(-N // (256 // nmat)) * -(-M // (64 * (kind - 3)))
        whole = (tiles * ks - groups) // (ks - 1)
    return kind, ks, groups, kb, inside, whole


def test_plan_shapes_reach_every_kernel(pkg):
    got = set()
    for nmat, M, N, K in PLAN_SHAPES:
        kind, ks, _, _, inside, whole = _plan(pkg, nmat, M, N, K)
        got.add((nmat, kind, ks > 1, whole > 0, (8 if N <= 8192 else 4) if inside else 0))
    want = {(n, k, False, False, 0) for n in (1, 2) for k in (0, 1, 2, 3, 4, 5, 8) if (n, k) not in ((2, 1), (2, 3))}
    want |= {(n, k, True, False, 0) for n in (1, 2) for k in (4, 5)} | {(n, 5, True, True, 0) for n in (1, 2)}
    want |= {(n, 8, False, False, w) for n in (1, 2) for w in (4, 8)}
    assert got == want, (got ^ want)


@pytest.mark.parametrize("nmat", [1, 2])
def test_plans_cover_the_outputs_and_fit(pkg, nmat):
    for cus in (256, 304, 64, 1):
        for N, K in ((5120, 17408), (17408, 5120), (1, 32), (33, 288), (1000, 1 << 20), (1 << 20, 64)):
            for M in (*range(1, 70), 100, 129, 256, 777, 1024, 1025, 2048, 65536):
                kind, ks, groups, kb, inside, whole = _plan(pkg, nmat, M, N, K, cus)
                units, feats = -(-K // 256), 256 // nmat if kind in (4, 5) else 32
                toks = {4: 64, 5: 128, 3: 64}.get(kind, 32)
                tiles = -(-N // feats) * -(-M // toks)
                assert whole in (0, tiles // cus * cus) and whole < tiles or ks == 1
                assert groups == whole + (tiles - whole) * ks and 1 <= ks <= units and (kind in (4, 5) or ks == 1)
                assert kb * 1024 == ((tiles - whole) * ks * 256 * toks * 4 if ks > 1 else 0) <= 64 << 20
                assert (kind == 8) == (M <= 16) and (kind not in (4, 5) or M > 32) and (kind != 3 or (M > 32 and nmat == 1))
                assert inside == (M <= 4 and M * units <= 68)
    out = (ctypes.c_int * 5)()
    for bad in ((0, 256, 256, 1, 256), (1, 0, 256, 1, 256), (1, 256, 48, 1, 256), (1, 256, 256, 3, 256), (1, 256, 256, 1, 0)):
        assert pkg.lib().qmlp_w4a8_plan(*bad, out) == E_SHAPE
    assert pkg.lib().qmlp_w4a8_plan(1, 256, 256, 1, 256, None) == E_NULL


# ---------------------------------------------------------------- refusals of the C entry points


def P(at):
    return ctypes.c_void_p(at)


X, W0, W1, RES, OUT, WS, GA, UA = (P(1 << k) for k in range(32, 40))
BIG = 1 << 31


def _linear(lib, x=X, xt=0, xs=256, w=W0, res=None, out=OUT, ws=WS, wsb=BIG, M=4, N=64, K=256, flags=0):
    return lib.qmlp_w4a8_linear(x, xt, xs, w, res, out, ws, wsb, M, N, K, flags, None)


def _swiglu(lib, x=X, xt=0, xs=256, w=W0, w1=W1, ga=None, ua=None, out=OUT, ws=WS, wsb=BIG, M=4, N=256, K=256, flags=0):
    return lib.qmlp_w4a8_swiglu(x, xt, xs, w, w1, ga, ua, out, ws, wsb, M, N, K, flags, None)


@pytest.mark.parametrize("call", [_linear, _swiglu])
def test_product_refusals(pkg, call):
    lib = pkg.lib()
    for arg in ("x", "w", "out"):
        assert call(lib, **{arg: None}) == E_NULL
    for arg in ("x", "w", "out", "ws"):
        assert call(lib, **{arg: P((1 << 41) + 8)}) == E_ALIGN
    for kw in ({"M": 0}, {"M": -1}, {"M": 65537}, {"N": 0}, {"N": -3}, {"K": 0}, {"K": 48}, {"N": 1 << 21},
               {"K": 1 << 21, "xs": 1 << 21}):
        assert call(lib, **kw) == E_SHAPE, kw
    assert call(lib, xt=3) == E_FORMAT and call(lib, xt=5) == E_FORMAT and call(lib, xt=-1) == E_FORMAT
    assert call(lib, flags=4) == E_FORMAT and call(lib, flags=16) == E_FORMAT
    for kw in ({"xs": 255}, {"xs": 260}, {"xs": -256}, {"xs": 258, "xt": 2}, {"xs": 1 << 50}):
        assert call(lib, **kw) == E_SHAPE, kw
    assert b"stride" in lib.qmlp_last_error()
    need = lib.qmlp_w4a8_workspace_bytes(40, 256 if call is _swiglu else 64, 256, 0)
    assert call(lib, wsb=need - 1, M=40) == E_WORKSPACE and call(lib, ws=None, M=40) == E_NULL
    assert call(lib, out=X) == E_SHAPE and call(lib, out=W0) == E_SHAPE
    assert call(lib, xs=1 << 20, out=P((1 << 32) + 3 * (2 << 20) + 16)) == E_SHAPE
    assert all(call(lib, ws=at, M=40) == E_SHAPE for at in (X, OUT, W0))
    assert call(lib, xt=4, out=X) == E_SHAPE and call(lib, xt=4, out=P((1 << 32) + 8400)) == E_SHAPE


def test_linear_residual_refusals(pkg):
    lib = pkg.lib()
    assert _linear(lib, res=P((1 << 41) + 4)) == E_ALIGN
    assert _linear(lib, res=P((1 << 36) + 64)) == E_SHAPE           # partly on out
    assert _linear(lib, res=OUT, flags=1) == E_SHAPE                # in place, out fp32 and residual bf16
    assert _linear(lib, res=OUT, flags=2) == E_SHAPE
    assert b"dtype" in lib.qmlp_last_error()
    assert _linear(lib, res=WS, M=40) == E_SHAPE
    assert _linear(lib, flags=8) == E_FORMAT                        # a packed output is the gate/up pair's


def test_swiglu_refusals(pkg):
    lib = pkg.lib()
    assert _swiglu(lib, w1=None) == E_NULL and _swiglu(lib, w1=P((1 << 41) + 8)) == E_ALIGN
    assert _swiglu(lib, out=W1) == E_SHAPE
    assert _swiglu(lib, flags=9) == E_FORMAT and _swiglu(lib, flags=2) == E_FORMAT
    assert _swiglu(lib, flags=8, N=288) == E_SHAPE
    assert b"256" in lib.qmlp_last_error()
    for arg in ("ga", "ua"):
        assert _swiglu(lib, **{arg: P((1 << 41) + 8)}) == E_ALIGN
        assert _swiglu(lib, **{arg: OUT}) == E_SHAPE and _swiglu(lib, **{arg: WS}, M=40) == E_SHAPE
        assert _swiglu(lib, **{arg: P((1 << 36) - 4 * 256 * 4 + 16)}) == E_SHAPE  # its last bytes on out


def test_quantize_refusals(pkg):
    lib = pkg.lib()
    n = omi.packed_bytes(4, 256)

    def q(x=X, xt=0, xs=256, rows=4, cols=256, packed=OUT, nbytes=n):
        return lib.qmlp_mxint8_quantize(x, xt, xs, rows, cols, packed, nbytes, None)

    assert q(x=None) == E_NULL and q(packed=None) == E_NULL and q(packed=P((1 << 36) + 8)) == E_ALIGN
    for kw in ({"rows": 0}, {"cols": 16}, {"cols": 0}, {"rows": 1 << 21}, {"xs": 200}, {"xs": 258, "xt": 2}):
        assert q(**kw) == E_SHAPE, kw
    assert q(nbytes=n - 1) == E_WORKSPACE and q(packed=X) == E_SHAPE and q(xt=3) == E_FORMAT and q(xt=4) == E_FORMAT

    def d(packed=X, rows=4, cols=256, out=OUT, ot=0):
        return lib.qmlp_mxint8_dequantize(packed, rows, cols, out, ot, None)

    assert d(packed=None) == E_NULL and d(out=None) == E_NULL and d(ot=1) == E_FORMAT and d(ot=4) == E_FORMAT
    assert d(rows=0) == E_SHAPE and d(cols=40) == E_SHAPE and d(out=X) == E_SHAPE and d(out=P((1 << 36) + 8)) == E_ALIGN

    def u(packed=X, rows=4, cols=256, q=OUT, scales=WS):
        return lib.qmlp_mxint8_unpack(packed, rows, cols, q, scales, None)

    assert u(packed=None) == E_NULL and u(q=None) == E_NULL and u(scales=None) == E_NULL
    assert u(rows=0) == E_SHAPE and u(cols=40) == E_SHAPE and u(q=X) == E_SHAPE and u(scales=X) == E_SHAPE
    assert u(scales=OUT) == E_SHAPE and u(q=P((1 << 36) + 8)) == E_ALIGN


def test_add_rmsnorm_refusals(pkg):
    lib = pkg.lib()
    nbytes = omi.packed_bytes(4, 256)

    def f(x=X, xt=0, xs=256, r=RES, rt=0, rs=256, w=W0, eps=1e-6, rows=4, cols=256, h=OUT, hs=256, n=GA, packed=UA,
          nb=nbytes):
        return lib.qmlp_add_rmsnorm(x, xt, xs, r, rt, rs, w, eps, rows, cols, h, hs, n, packed, nb, None)

    for kw in ({"x": None}, {"w": None}, {"h": None}, {"n": None, "packed": None}, {"r": None}):
        assert f(**kw) == E_NULL, kw
    for arg in ("x", "r", "w", "h", "n", "packed"):
        assert f(**{arg: P((1 << 41) + 8)}) == E_ALIGN, arg
    for kw in ({"rows": 0}, {"cols": 48}, {"cols": 0}, {"xs": 255}, {"rs": 248}, {"hs": 250}, {"rt": 2, "rs": 258},
               {"eps": -1.0}, {"eps": float("nan")}):
        assert f(**kw) == E_SHAPE, kw
    assert f(xt=1) == E_FORMAT and f(rt=1) == E_FORMAT and f(xt=4) == E_FORMAT and f(rt=3) == E_FORMAT
    assert f(nb=nbytes - 1) == E_WORKSPACE
    for kw in ({"h": X}, {"n": X}, {"packed": X}, {"n": RES}, {"packed": RES}, {"h": W0}, {"n": W0}, {"packed": W0},
               {"n": OUT}, {"packed": OUT}, {"packed": GA}, {"h": P((1 << 35) + 16)}, {"h": RES, "hs": 264}):
        assert f(**kw) == E_SHAPE, kw


# ---------------------------------------------------------------- refusals of the Python entry points


def test_python_refusals_need_no_gpu(pkg):
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    w = pkg.PackedWeight(torch.zeros(8, dtype=torch.uint8), 64, 256, "mxfp4")
    t = pkg.Mx8Tensor(torch.zeros(8448, dtype=torch.uint8), 4, 256)
    for f in (lambda: pkg.quantize_mxint8(x), lambda: pkg.w4a8_linear(x, w), lambda: pkg.w4a8_swiglu(x, w, w),
              lambda: pkg.w4a8_linear(t, w), lambda: pkg.dequantize(t), lambda: pkg.unpack_canonical(t),
              lambda: pkg.add_rmsnorm(x, x, x[0])):
        with pytest.raises(ValueError, match="GPU"):
            f()
    with pytest.raises(ValueError, match="output"):
        pkg.add_rmsnorm(x, x, x[0], output="mxfp4")
    for bad in (None, [1.0], t):
        with pytest.raises(ValueError):
            pkg.quantize_mxint8(bad)
    with pytest.raises(ValueError):
        pkg.w4a8_linear(pkg.MxTensor(torch.zeros(8, dtype=torch.uint8), 4, 256), w)
    with pytest.raises(ValueError):
        pkg.mxfp4_linear(t, w)
