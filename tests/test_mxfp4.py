"""MXFP4 without a GPU: the oracle's format, buffer sizes, and every refusal of the entry points (made
before a device is touched)."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

from oracle import mxfp4 as omx

E_SHAPE, E_ALIGN, E_FORMAT, E_WORKSPACE, E_NULL = -1, -2, -3, -5, -6


# ---------------------------------------------------------------- the oracle


def test_codes_are_nearest_with_ties_to_even():
    v = np.array([0.0, 0.25, 0.2500001, 0.5, 0.75, 0.7499999, 1.25, 1.2500001, 1.75, 2.5, 2.6, 3.5, 3.4, 5.0, 5.1, 6.0, 7.9])
    want = [0, 0, 1, 1, 2, 1, 2, 3, 4, 4, 5, 6, 5, 6, 7, 7, 7]
    assert omx.nearest_codes(v).tolist() == want
    assert omx.nearest_codes(-v).tolist() == [c + 8 for c in want]


def test_every_representable_block_comes_back():
    """A block whose largest magnitude is 4 or 6 times its scale is its own quantisation."""
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 16, (64, 96), dtype=np.uint8)
    codes[:, ::32] = rng.choice([6, 7, 14, 15], (64, 3))
    scales = rng.integers(1, 253, (64, 3), dtype=np.uint8)
    c, s = omx.quantize(omx.dequantize(codes, scales))
    assert np.array_equal(c, codes) and np.array_equal(s, scales)


def test_quantize_edges():
    x = np.zeros((6, 32))
    x[1, 3], x[2, 5] = np.inf, np.nan
    x[3, 0], x[3, 1] = 7.99, -3.0            # saturates at 6 times 2^0
    x[4, 0] = 2.0 ** -130                    # below the smallest scale's steps: 2^-130 / 2^-126 = 1/16
    x[5, 0], x[5, 1] = 3.4028234663852886e38, 2.0 ** -149
    codes, scales = omx.quantize(x)
    assert scales[:, 0].tolist() == [1, 255, 255, 127, 1, 252]
    assert not codes[0].any() and not codes[1].any() and not codes[4].any()
    assert codes[3, :2].tolist() == [7, 13] and codes[5, :2].tolist() == [7, 0]
    d = omx.dequantize(codes, scales)
    assert np.isnan(d[1]).all() and np.isnan(d[2]).all() and d[3, 0] == 6.0


def test_pack_places_each_block():
    rng = np.random.default_rng(1)
    codes = rng.integers(0, 16, (33, 288), dtype=np.uint8)
    scales = rng.integers(0, 255, (33, 9), dtype=np.uint8)
    p = omx.pack(codes, scales)
    assert p.size == omx.packed_bytes(33, 288) == 4 * 4352 + 256
    # row 32, block 8: unit (1, 1), its first chunk and first scale byte
    at = 3 * 4352
    assert np.array_equal(p[at:at + 16], omx.join(codes[32:33, 256:288])[0]) and p[at + 4096] == scales[32, 8]
    # row 5, block 3: dword 5 + 32, byte 1
    assert p[4096 + 4 * 37 + 1] == scales[5, 3]
    assert np.array_equal(p[(3 * 32 + 5) * 16:(3 * 32 + 5) * 16 + 16], omx.join(codes[5:6, 96:128])[0])
    assert np.array_equal(omx.split(omx.join(codes)), codes)


# ---------------------------------------------------------------- sizes


@pytest.mark.parametrize("rows,cols", [(1, 32), (32, 256), (33, 288), (17408, 5120), (5120, 17408), (777, 1056)])
def test_packed_bytes(pkg, rows, cols):
    assert pkg.lib().qmlp_packed_bytes(rows, cols, pkg.FMT_MXFP4) == omx.packed_bytes(rows, cols)


def test_packed_bytes_refuses(pkg):
    for rows, cols in ((0, 32), (1, 16), (1, 0), (1, 33), (-1, 32), (1 << 21, 32), (1, 1 << 21)):
        assert pkg.lib().qmlp_packed_bytes(rows, cols, pkg.FMT_MXFP4) == 0


def test_workspaces_never_shrink_as_m_grows(pkg):
    lib = pkg.lib()
    Ms = list(range(1, 700)) + [1023, 1024, 2047, 2048, 2049, 65536]
    for N, K in ((5120, 17408), (17408, 5120), (100, 32), (1, 1056)):
        for x_type in range(4):
            sizes = [lib.qmlp_mx_workspace_bytes(M, N, K, x_type) for M in Ms]
            assert sizes[Ms.index(33)] > 0 and sizes == sorted(sizes)
            assert (sizes[Ms.index(32)] == 0) == (x_type == 3)
    for H, I in ((5120, 17408), (256, 256)):
        sizes = [lib.qmlp_workspace_bytes(M, H, I, pkg.FMT_MXFP4) for M in Ms]
        assert sizes[0] > 0 and sizes == sorted(sizes)
    assert lib.qmlp_workspace_bytes(16, 5120 + 32, 17408, pkg.FMT_MXFP4) == 0  # the block's sizes: multiples of 256
    for bad in ((0, 256, 256), (65537, 256, 256), (1, 0, 256), (1, 256, 48)):
        assert lib.qmlp_mx_workspace_bytes(*bad, 0) == 0
    # a 16-token forward fits the library's own scratch
    assert lib.qmlp_workspace_bytes(32, 5120, 17408, pkg.FMT_MXFP4) <= 33554432


# ---------------------------------------------------------------- plans

# (matrices, M, N, K): sizes whose plans take every kernel that the products launch, whole and with the K
# range in pieces, and quantise inside and in front; the GPU tests run them all.
PLAN_SHAPES = [(1, 5, 65, 96), (1, 1, 65, 96), (1, 5, 8438, 1088), (1, 2, 8222, 1056), (1, 5, 71, 1056),
               (1, 1, 65, 1088), (1, 4, 300, 8480), (1, 33, 4279, 1088), (1, 1107, 65, 96), (1, 1097, 66, 3904),
               (1, 33, 70, 30112), (1, 2311, 1592, 96), (1, 1392, 76, 33632), (1, 257, 5120, 17440), (1, 1688, 4747, 96),
               (1, 1361, 8237, 96), (1, 2047, 5125, 1120), (2, 5, 8448, 96), (2, 1, 8448, 96), (2, 5, 256, 96),
               (2, 1, 256, 96), (2, 33, 4864, 2336), (2, 1025, 256, 96), (2, 33, 256, 22816), (2, 1635, 1280, 96),
               (2, 65, 2816, 16352), (2, 1178, 3328, 96), (2, 782, 6912, 96), (2, 777, 3328, 1056)]


def _plan(pkg, nmat, M, N, K, cus=256):
    out = (ctypes.c_int * 5)()
    assert pkg.lib().qmlp_mx_plan(M, N, K, nmat, cus, out) == 0
    return list(out)


def test_plan_shapes_reach_every_kernel(pkg):
    got = set()
    for nmat, M, N, K in PLAN_SHAPES:
        kind, ks, _, _, inside = _plan(pkg, nmat, M, N, K)
        got.add((nmat, kind, ks > 1, inside))
    want = {(n, k, False, 0) for n in (1, 2) for k in range(8) if (n, k) != (2, 1)}
    want |= {(n, k, True, 0) for n in (1, 2) for k in (4, 5)}
    want |= {(1, 0, False, 1), (1, 1, False, 1), (1, 2, False, 1), (2, 0, False, 1), (2, 2, False, 1)}
    assert got == want


@pytest.mark.parametrize("nmat", [1, 2])
def test_plans_cover_the_outputs_and_fit(pkg, nmat):
    for cus in (256, 304, 64, 1):
        for N, K in ((5120, 17408), (17408, 5120), (1, 32), (33, 288), (1000, 1 << 20), (1 << 20, 64)):
            for M in (*range(1, 70), 100, 129, 256, 777, 1024, 1025, 2048, 65536):
                kind, ks, groups, kb, inside = _plan(pkg, nmat, M, N, K, cus)
                units, feats = -(-K // 256), 32 if kind < 4 else 256 // nmat
                toks = 64 * (kind - 3) if kind > 3 else 64 if kind == 3 else 32
                tiles = -(-N // feats) * -(-M // toks)
                assert groups == tiles * ks and 1 <= ks <= units and (kind in (4, 5) or ks == 1)
                assert kb * 1024 == (tiles * ks * 256 * toks * 4 if ks > 1 else 0) <= 64 << 20
                assert kind < 4 or M > 32
                assert inside == (M <= 4 and M * units <= 136) and not (inside and kind > 2)
    out = (ctypes.c_int * 5)()
    for bad in ((0, 256, 256, 1, 256), (1, 0, 256, 1, 256), (1, 256, 48, 1, 256), (1, 256, 256, 3, 256), (1, 256, 256, 1, 0)):
        assert pkg.lib().qmlp_mx_plan(*bad, out) == E_SHAPE
    assert pkg.lib().qmlp_mx_plan(1, 256, 256, 1, 256, None) == E_NULL


# ---------------------------------------------------------------- refusals of the C entry points


def P(at):
    return ctypes.c_void_p(at)


X, W0, W1, RES, OUT, WS = (P(1 << k) for k in range(32, 38))
BIG = 1 << 31


def _linear(lib, x=X, xt=0, xs=256, w=W0, res=None, out=OUT, ws=WS, wsb=BIG, M=4, N=64, K=256, flags=0):
    return lib.qmlp_mx_linear(x, xt, xs, w, res, out, ws, wsb, M, N, K, flags, None)


def _swiglu(lib, x=X, xt=0, xs=256, w=W0, w1=W1, out=OUT, ws=WS, wsb=BIG, M=4, N=256, K=256, flags=0):
    return lib.qmlp_mx_swiglu(x, xt, xs, w, w1, out, ws, wsb, M, N, K, flags, None)


@pytest.mark.parametrize("call", [_linear, _swiglu])
def test_product_refusals(pkg, call):
    lib = pkg.lib()
    for arg in ("x", "w", "out"):
        assert call(lib, **{arg: None}) == E_NULL
    for arg in ("x", "w", "out", "ws"):
        assert call(lib, **{arg: P((1 << 40) + 8)}) == E_ALIGN
    for kw in ({"M": 0}, {"M": -1}, {"M": 65537}, {"N": 0}, {"N": -3}, {"K": 0}, {"K": 48}, {"N": 1 << 21},
               {"K": 1 << 21, "xs": 1 << 21}):
        assert call(lib, **kw) == E_SHAPE, kw
    assert call(lib, xt=4) == E_FORMAT and call(lib, xt=-1) == E_FORMAT
    assert call(lib, flags=8) == E_FORMAT
    for kw in ({"xs": 255}, {"xs": 260}, {"xs": -256}, {"xs": 258, "xt": 2}, {"xs": 1 << 50}):
        assert call(lib, **kw) == E_SHAPE, kw
    assert b"stride" in lib.qmlp_last_error()
    need = lib.qmlp_mx_workspace_bytes(40, 256 if call is _swiglu else 64, 256, 0)
    assert call(lib, wsb=need - 1, M=40) == E_WORKSPACE and call(lib, ws=None, M=40) == E_NULL
    # out on x, on a weight, on the last strided row of x; the workspace on an argument
    assert call(lib, out=X) == E_SHAPE and call(lib, out=W0) == E_SHAPE
    assert call(lib, xs=1 << 20, out=P((1 << 32) + 3 * (2 << 20) + 16)) == E_SHAPE
    assert all(call(lib, ws=at, M=40) == E_SHAPE for at in (X, OUT, W0))
    assert call(lib, xt=3, out=X) == E_SHAPE


def test_linear_residual_refusals(pkg):
    lib = pkg.lib()
    assert _linear(lib, res=P((1 << 40) + 4)) == E_ALIGN
    assert _linear(lib, res=P((1 << 36) + 64)) == E_SHAPE           # partly on out
    assert _linear(lib, res=OUT, flags=1) == E_SHAPE                # in place, out fp32 and residual bf16
    assert _linear(lib, res=OUT, flags=2) == E_SHAPE
    assert b"dtype" in lib.qmlp_last_error()
    assert _linear(lib, res=WS, M=40) == E_SHAPE
    assert _linear(lib, flags=4) == E_FORMAT                        # a packed output is the gate/up pair's


def test_swiglu_refusals(pkg):
    lib = pkg.lib()
    assert _swiglu(lib, w1=None) == E_NULL and _swiglu(lib, w1=P((1 << 40) + 8)) == E_ALIGN
    assert _swiglu(lib, out=W1) == E_SHAPE
    assert _swiglu(lib, flags=5) == E_FORMAT and _swiglu(lib, flags=2) == E_FORMAT
    assert _swiglu(lib, flags=4, N=288) == E_SHAPE
    assert b"256" in lib.qmlp_last_error()


def test_quantize_and_dequantize_refusals(pkg):
    lib = pkg.lib()
    n = omx.packed_bytes(4, 256)

    def q(x=X, xt=0, xs=256, rows=4, cols=256, packed=OUT, nbytes=n):
        return lib.qmlp_mx_quantize(x, xt, xs, rows, cols, packed, nbytes, None)

    def norm(h=X, hs=256, w=W0, eps=1e-6, rows=4, cols=256, packed=OUT, nbytes=n):
        return lib.qmlp_mx_quantize_rmsnorm(h, hs, w, eps, rows, cols, packed, nbytes, None)

    for f in (q, norm):
        first = {"x": None} if f is q else {"h": None}
        assert f(**first) == E_NULL and f(packed=None) == E_NULL and f(packed=P((1 << 36) + 8)) == E_ALIGN
        for kw in ({"rows": 0}, {"cols": 16}, {"cols": 0}, {"rows": 1 << 21}):
            assert f(**kw) == E_SHAPE
        assert f(nbytes=4351) == E_WORKSPACE and f(packed=X) == E_SHAPE
    assert q(xt=3) == E_FORMAT and q(xt=2, xs=258) == E_SHAPE and q(xs=200) == E_SHAPE
    assert norm(w=None) == E_NULL and norm(w=P((1 << 33) + 2)) == E_ALIGN and norm(packed=W0) == E_SHAPE
    for eps in (-1.0, float("nan")):
        assert norm(eps=eps) == E_SHAPE

    def d(packed=X, rows=4, cols=256, out=OUT, ot=0):
        return lib.qmlp_mx_dequantize(packed, rows, cols, out, ot, None)

    assert d(packed=None) == E_NULL and d(out=None) == E_NULL and d(ot=1) == E_FORMAT and d(ot=3) == E_FORMAT
    assert d(rows=0) == E_SHAPE and d(cols=40) == E_SHAPE and d(out=X) == E_SHAPE and d(out=P((1 << 36) + 8)) == E_ALIGN


def test_format_entry_points_take_the_format(pkg):
    lib, F = pkg.lib(), pkg.FMT_MXFP4
    assert lib.qmlp_pack(X, None, 3, 32, F, OUT, 1 << 20, None) == E_NULL
    assert lib.qmlp_pack(X, W0, 3, 48, F, OUT, 1 << 20, None) == E_SHAPE
    assert b"32" in lib.qmlp_last_error()
    assert lib.qmlp_pack(X, W0, 3, 32, F, OUT, 4607, None) == E_WORKSPACE
    assert lib.qmlp_quantize_pack(X, 3, 48, F, OUT, 1 << 20, None) == E_SHAPE
    assert lib.qmlp_quantize_pack(X, 3, 32, F, OUT, 4607, None) == E_WORKSPACE
    assert lib.qmlp_unpack_mxfp4(X, 0, 32, W0, W1, None) == E_SHAPE
    out8 = (ctypes.c_int * 8)()
    assert lib.qmlp_plan_tiles(64, 256, 256, F, 0, 256, out8) == E_SHAPE  # the tile plans are the other formats'
    # the forward: a workspace that is too small, sizes that are not multiples of 256, an overlap
    need = lib.qmlp_workspace_bytes(4, 256, 512, F)
    assert lib.qmlp_forward(X, W0, W1, W0, None, OUT, WS, need - 1, 4, 256, 512, F, None) == E_WORKSPACE
    assert lib.qmlp_forward(X, W0, W1, W0, None, OUT, WS, BIG, 4, 288, 512, F, None) == E_SHAPE
    assert lib.qmlp_forward(X, W0, W1, W0, None, X, WS, BIG, 4, 256, 512, F, None) == E_SHAPE


# ---------------------------------------------------------------- refusals of the Python entry points


def test_python_refusals_need_no_gpu(pkg):
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    w = pkg.PackedWeight(torch.zeros(8, dtype=torch.uint8), 64, 256, "mxfp4")
    for f in (lambda a: pkg.quantize_mxfp4(a), lambda a: pkg.mxfp4_linear(a, w), lambda a: pkg.mxfp4_swiglu(a, w, w)):
        with pytest.raises(ValueError, match="GPU"):
            f(x)
        with pytest.raises(ValueError, match="Tensor"):
            f([1.0])
    t = pkg.MxTensor(torch.zeros(8, dtype=torch.uint8), 4, 256)
    for bad in (pkg.PackedWeight(w.buf, 64, 256, "bfp8"), t, w.buf):
        with pytest.raises(ValueError, match="mxfp4"):
            pkg.mxfp4_linear(t, bad)
    with pytest.raises(ValueError, match="columns"):
        pkg.mxfp4_linear(t, pkg.PackedWeight(w.buf, 64, 288, "mxfp4"))
    with pytest.raises(ValueError, match="rows"):
        pkg.mxfp4_swiglu(t, w, pkg.PackedWeight(w.buf, 32, 256, "mxfp4"))
    with pytest.raises(ValueError, match="256"):
        pkg.mxfp4_swiglu(t, w, w, quantize=True)
    with pytest.raises(ValueError, match="quantize"):
        pkg.mxfp4_swiglu(t, w, w, quantize=True, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="out_dtype"):
        pkg.mxfp4_linear(t, w, out_dtype=torch.float16)
    for f in (pkg.dequantize, pkg.unpack_canonical, lambda v: pkg.mxfp4_linear(v, w),
              lambda v: pkg.mxfp4_swiglu(v, w, w)):  # host memory never reaches a kernel
        with pytest.raises(ValueError, match="GPU"):
            f(t)
    with pytest.raises(ValueError, match="dtype"):
        pkg.dequantize(t, dtype=torch.float16)
    with pytest.raises(ValueError, match="dtype"):
        pkg.dequantize(pkg.PackedWeight(w.buf, 64, 256, "bfp8"), dtype=torch.bfloat16)
    for q, e in itertools.product((x, torch.zeros(4, 128, dtype=torch.uint8)), repeat=2):
        with pytest.raises(ValueError):
            pkg.pack_canonical(q, e, "mxfp4")


def test_formats(pkg):
    assert pkg.matrix_formats("mxfp4") == ("mxfp4", "mxfp4") and "mxfp4" in pkg.WEIGHT_FORMATS
    w = pkg.PackedWeight(torch.zeros(8, dtype=torch.uint8), 64, 256, "mxfp4")
    assert w.stream_bytes == 64 * 256 * 17 // 32
    from qwen_mlp_amd import mlp

    mlp.check_formats(pkg.MLPWeights(w, w, w))
    with pytest.raises(ValueError, match="formats"):
        mlp.check_formats(pkg.MLPWeights(w, pkg.PackedWeight(w.buf, 64, 256, "bfp8"), w))


def test_a_stream_of_another_gpu_is_refused(pkg):
    from qwen_mlp_amd import _lib

    class Stream:
        device = torch.device("cuda", 1)

    with pytest.raises(ValueError, match="cuda:1"):
        _lib.on_device(torch.device("cuda", 0), Stream())


def test_workload_bytes_of_every_format(pkg):
    """A workload's weight bytes are those that the packed matrices' kernels stream."""
    from qwen_mlp_amd import workloads

    for fmt in pkg.WEIGHT_FORMATS:
        wl = workloads.Workload("any", 512, 1024, 16, fmt, False)
        gate_up, down = (pkg.PackedWeight(None, 512, 1024, f) for f in pkg.matrix_formats(fmt))
        assert wl.weight_bytes() == 2 * gate_up.stream_bytes + down.stream_bytes
        assert wl.algorithmic_bytes() == wl.weight_bytes() + 4 * 16 * 512


def test_the_block_takes_activations_beyond_32_bit_offsets(pkg):
    """As its products do: the last refusal before a device is touched is the workspace's."""
    lib, F = pkg.lib(), pkg.FMT_MXFP4
    for M, H, I in ((65536, 256, 16640), (65536, 5120, 17408), (65536, 16640, 256)):
        need = lib.qmlp_workspace_bytes(M, H, I, F)
        assert need > 0
        assert lib.qmlp_forward(P(1 << 40), W0, W1, W0, None, P(1 << 42), P(1 << 44), need - 1, M, H, I, F, None) == E_WORKSPACE
        assert lib.qmlp_forward_rmsnorm(P(1 << 40), W0, 1e-6, W0, W1, W0, P(1 << 42), P(1 << 44), need - 1, M, H, I, F, 0,
                                        None) == E_WORKSPACE


# The tiled kernels, with the last tile of features full and part full (a row length that is not a multiple of
# 4 among them), whole and in pieces; tests/test_gpu_mxfp4_tiles.py runs them.
TILE_SHAPES = [(1, 1107, 256, 96), (1, 1107, 65, 96), (1, 1097, 256, 3904), (1, 1097, 66, 3904),
               (1, 1688, 4608, 96), (1, 2311, 1593, 96), (1, 1392, 256, 33632), (1, 1392, 77, 33632),
               (1, 2047, 4608, 96), (1, 2047, 4618, 96), (1, 2047, 6144, 96), (1, 1361, 8237, 96),
               (2, 1025, 256, 96), (2, 1025, 250, 96), (2, 33, 256, 22816), (2, 33, 250, 22816),
               (2, 1635, 1280, 96), (2, 1635, 1275, 96), (2, 65, 2816, 16352), (2, 777, 2819, 1056),
               (2, 65, 2803, 16352), (2, 1178, 3328, 96), (2, 1178, 3331, 96), (2, 782, 6912, 96), (2, 782, 6915, 96)]


def tile_plan(pkg, nmat, M, N, K):
    """(tile height in units of 64 tokens, pieces of K) of a product that is planned on tiles."""
    kind, ks, *_ = _plan(pkg, nmat, M, N, K)
    assert kind >= 4, f"{nmat} x {M} x {N} x {K} is not planned on tiles"
    return kind - 3, ks


def test_tile_shapes_reach_every_tiled_kernel(pkg):
    got = {(n, *tile_plan(pkg, n, M, N, K), N % (256 // n) == 0) for n, M, N, K in TILE_SHAPES}
    got = {(n, h, ks > 1, full) for n, h, ks, full in got}
    heights = [(h, False) for h in (1, 2, 3, 4)] + [(h, True) for h in (1, 2)]
    assert got == {(n, h, split, full) for n in (1, 2) for h, split in heights for full in (True, False)}
    for n in (1, 2):  # rows that start misaligned for vector stores, whole and in pieces
        odd = {tile_plan(pkg, n, M, N, K)[1] > 1 for m, M, N, K in TILE_SHAPES if m == n and N % 4}
        assert odd == {True, False}
