"""MXFP4 on the GPU against the oracle's definition in 64 bits.

Quantisation, packing and dequantisation are compared bit for bit.  A product's operands are small
multiples of powers of two, so every single product is exact and only the fp32 sums round: the
matrix cores take K in steps of 64, each step rounds at most twice (its own sum of 64 products, then
the accumulator), each by at most 2^-23 of the magnitudes summed so far, and splitting K over waves
or pieces adds at most 32 more additions.  ``_sum_error`` is that bound; an output's own rounding to
bf16 comes on top (half a step, at most 2^-8 of the value)."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as omx
from test_mxfp4 import PLAN_SHAPES

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _sum_error(K, magnitudes):
    return (2 * (K / 64 + 1) + 32) * 2.0 ** -23 * magnitudes


def _bf16_error(y, err):
    """Bound of |bf16(y') - y| for |y' - y| <= err: half a step of 8 significant bits on top."""
    return err + 2.0 ** -8 * (np.abs(y) + err)


def _rows(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * scale
    x *= torch.exp2(torch.randint(-6, 7, (rows, cols // 32, 1), generator=g).float()).expand(-1, -1, 32).reshape(rows, cols)
    return x.to(dtype)


def _np(t):
    return t.double().cpu().numpy()


def _unpack(pkg, t):
    q, e = pkg.unpack_canonical(t)
    return omx.split(q.cpu().numpy()), e.cpu().numpy()


def _weight(pkg, rows, cols, seed, device):
    """A packed weight and its dequantised values, from random codes and scales."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    scales = rng.integers(117, 125, (rows, cols // 32), dtype=np.uint8)
    pw = pkg.pack_canonical(torch.from_numpy(omx.join(codes)).to(device), torch.from_numpy(scales).to(device), "mxfp4")
    return pw, omx.dequantize(codes, scales)


# ---------------------------------------------------------------- the format


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 5120), (3, 64), (8, 256), (9, 288), (33, 224), (257, 1056),
                                       (1030, 8320)])
def test_quantize_is_the_definition(pkg, cuda, rows, cols, dtype):
    print(f"case quantize {rows}x{cols} {dtype}", flush=True)
    x = _rows(rows, cols, dtype, rows + cols)
    t = pkg.quantize_mxfp4(x.to(cuda))
    assert t.shape == (rows, cols) and t.buf.numel() == omx.packed_bytes(rows, cols)
    codes, scales = _unpack(pkg, t)
    want, wants = omx.quantize(x.double().numpy())
    assert np.array_equal(scales, wants) and np.array_equal(codes, want)
    d = omx.dequantize(want, wants)
    for dt in (torch.float32, torch.bfloat16):
        assert np.array_equal(_np(pkg.dequantize(t, dtype=dt)), d)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_every_16_bit_value_and_special_blocks(pkg, cuda, dtype):
    """Every bf16 / fp16 bit pattern (as fp32 too) beside block maxima of every binade; infinities and NaN."""
    if dtype == torch.float32:
        x = torch.arange(65536, dtype=torch.int32).mul(65536).add(0x5a5a).view(torch.float32)
    else:
        x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x.reshape(-1, 32)
    shuffled = x.reshape(-1)[torch.randperm(65536, generator=torch.Generator().manual_seed(7))].reshape(-1, 32)
    finite = torch.nan_to_num(shuffled.float(), nan=1.0, posinf=2.0, neginf=-2.0).to(dtype)
    x = torch.cat([x, shuffled, finite, torch.zeros(8, 32, dtype=dtype)])
    codes, scales = _unpack(pkg, pkg.quantize_mxfp4(x.to(cuda)))
    want, wants = omx.quantize(x.double().numpy())
    assert np.array_equal(scales, wants) and np.array_equal(codes, want)


def test_quantize_strided_rows(pkg, cuda):
    for dtype, pad in ((torch.bfloat16, 8), (torch.float32, 4), (torch.float16, 40)):
        wide = _rows(21, 160, dtype, 3).to(cuda)
        wide = torch.cat([wide, torch.full((21, pad), float("nan"), dtype=dtype, device=cuda)], dim=1)
        x = wide[:, :160]
        assert not x.is_contiguous()
        a, b = pkg.quantize_mxfp4(x), pkg.quantize_mxfp4(x.contiguous())
        for u, v in zip(pkg.unpack_canonical(a), pkg.unpack_canonical(b)):
            assert torch.equal(u, v)
    for bad in (wide[:, 1:161], wide.T, wide[:, :160:2], wide[:, :16], wide[:0, :160], wide[0], wide.to(torch.float64)):
        with pytest.raises(ValueError):
            pkg.quantize_mxfp4(bad)


@pytest.mark.parametrize("rows,cols", [(1, 32), (31, 256), (32, 288), (70, 1024)])
def test_pack_layout_round_trip_and_weights(pkg, cuda, rows, cols):
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    scales = rng.integers(0, 255, (rows, cols // 32), dtype=np.uint8)
    q, e = torch.from_numpy(omx.join(codes)).to(cuda), torch.from_numpy(scales).to(cuda)
    pw = pkg.pack_canonical(q, e, "mxfp4")
    assert np.array_equal(pw.buf.cpu().numpy(), omx.pack(codes, scales))
    for a, b in zip(pkg.unpack_canonical(pw), (q, e)):
        assert torch.equal(a, b)
    with np.errstate(over="ignore"):
        d = omx.dequantize(codes, scales).astype(np.float32)
    assert np.array_equal(pkg.dequantize(pw).cpu().numpy(), d)
    assert np.array_equal(_np(pkg.dequantize(pw, dtype=torch.bfloat16)), d.astype(np.float64))
    # a bf16 weight: quantised and packed at once is the same as one after the other
    w = _rows(rows, cols, torch.bfloat16, 5, 0.02)
    pw = pkg.pack_weight(w.to(cuda), "mxfp4")
    assert np.array_equal(pw.buf.cpu().numpy(), omx.pack(*omx.quantize(w.double().numpy())))
    assert pw.max_row_norm == 0.0 and pw.flushed_groups == 0


def test_weights_that_are_not_numbers_are_refused(pkg, cuda):
    w = torch.ones(5, 64, dtype=torch.bfloat16, device=cuda)
    w[2, 40] = float("inf")
    with pytest.raises(ValueError, match="non-finite values in 1 groups"):
        pkg.pack_weight(w, "mxfp4")
    e = torch.full((5, 2), 120, dtype=torch.uint8, device=cuda)
    e[1] = 255
    with pytest.raises(ValueError, match="non-finite values in 2 groups"):
        pkg.pack_canonical(torch.zeros(5, 32, dtype=torch.uint8, device=cuda), e, "mxfp4")


@pytest.mark.parametrize("rows,cols", [(1, 5120), (16, 5120), (3, 32), (5, 288), (40, 8192), (2, 17408)])
def test_norm_in_front(pkg, cuda, rows, cols):
    """The blocks of bf16(rmsnorm(x) (1 + w)): where the norm's fp32 error (sums of squares of
    non-negative terms in at most cols / 2048 + 16 steps and a few operations, below 2^-19 of the value)
    cannot move a bf16 rounding of a block, the block is the oracle's."""
    x = _rows(rows, cols, torch.bfloat16, 11)
    w = (torch.randn(cols, generator=torch.Generator().manual_seed(2)) * 0.1).bfloat16()
    codes, scales = _unpack(pkg, pkg.quantize_mxfp4(x.to(cuda), norm_weight=w.to(cuda), eps=1e-6))
    d = x.double()
    n = d / torch.sqrt((d * d).mean(dim=1, keepdim=True) + 1e-6) * (1 + w.double())
    lo, hi = (n * (1 - 2.0 ** -19)).bfloat16(), (n * (1 + 2.0 ** -19)).bfloat16()
    sure = (lo == hi).reshape(rows, -1, 32).all(dim=2).numpy()
    want, wants = omx.quantize(lo.double().numpy())
    assert sure.mean() > 0.8  # a rounding border lies within 2^-19 of one value in 2^10 or so
    assert np.array_equal(scales[sure], wants[sure])
    assert np.array_equal(codes.reshape(rows, -1, 32)[sure], want.reshape(rows, -1, 32)[sure])
    # strided rows give the same bytes
    wide = torch.cat([x, x], dim=1).to(cuda)[:, :cols]
    for a, b in zip(pkg.unpack_canonical(pkg.quantize_mxfp4(wide, norm_weight=w.to(cuda))), (omx.join(codes), scales)):
        assert np.array_equal(a.cpu().numpy(), b)
    with pytest.raises(ValueError):
        pkg.quantize_mxfp4(x.to(cuda).float(), norm_weight=w.to(cuda))
    with pytest.raises(ValueError):
        pkg.quantize_mxfp4(x.to(cuda), norm_weight=w[1:].to(cuda))


# ---------------------------------------------------------------- the products

SHAPES = [(1, 1, 32), (1, 33, 64), (2, 100, 224), (5, 3, 1056), (16, 256, 288), (31, 31, 512), (32, 32, 256),
          (33, 64, 2080), (64, 1000, 96), (65, 130, 544), (100, 257, 1024), (128, 96, 4352), (257, 513, 800),
          (300, 1024, 256), (1, 5120, 5120), (4, 640, 17408), (17, 384, 8704), (513, 260, 2304), (1000, 300, 512)]


def _product_case(pkg, cuda, M, N, K, dtype, seed=0):
    x = _rows(M, K, dtype, M * 7 + K + seed)
    w, wd = _weight(pkg, N, K, N + K + seed, cuda)
    return x.to(cuda), omx.dequantize(*omx.quantize(x.double().numpy())), w, wd


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(pkg, cuda, M, N, K):
    print(f"case linear {M}x{N}x{K}", flush=True)
    x, xd, w, wd = _product_case(pkg, cuda, M, N, K, DTYPES[(M + N) % 3])
    ref, mag = omx.linear(xd, wd)
    err = _sum_error(K, mag)
    y = pkg.mxfp4_linear(x, w, out_dtype=torch.float32)
    assert y.shape == (M, N) and y.dtype == torch.float32
    assert (np.abs(_np(y) - ref) <= err).all()
    # the same from a packed activation, into a given output, twice: the same bits
    t = pkg.quantize_mxfp4(x)
    out = torch.full((M, N), 7.0, device=cuda)
    assert pkg.mxfp4_linear(t, w, out=out) is out and torch.equal(out, y)
    yb = pkg.mxfp4_linear(t, w)
    assert yb.dtype == torch.bfloat16 and torch.equal(yb, y.bfloat16())
    # residuals
    r = torch.randn(M, N, generator=torch.Generator().manual_seed(M)).to(cuda)
    y2 = pkg.mxfp4_linear(t, w, residual=r, out_dtype=torch.float32)
    full = ref + _np(r)
    assert (np.abs(_np(y2) - full) <= err + 2.0 ** -24 * (np.abs(full) + err)).all()
    rb = r.bfloat16()
    y3 = pkg.mxfp4_linear(x, w, residual=rb)
    full = ref + _np(rb)
    assert (np.abs(_np(y3) - full) <= _bf16_error(full, err * (1 + 2.0 ** -23))).all()
    inplace = rb.clone()
    assert torch.equal(pkg.mxfp4_linear(x, w, residual=inplace, out=inplace), y3)
    assert torch.equal(pkg.mxfp4_linear(t, w, residual=r, out=r), y2)


def _silu(g):
    return g / (1 + np.exp(-np.clip(g, -700, 700)))


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_swiglu(pkg, cuda, M, N, K):
    print(f"case swiglu {M}x{N}x{K}", flush=True)
    x, xd, w1, w1d = _product_case(pkg, cuda, M, N, K, DTYPES[(M + K) % 3])
    w3, w3d = _weight(pkg, N, K, 99, cuda)
    g, gm = omx.linear(xd, w1d)
    u, um = omx.linear(xd, w3d)
    ge, ue = _sum_error(K, gm), _sum_error(K, um)
    s = _silu(g)
    # |silu'| < 1.1; the kernel's exponential has a relative error of about |g| 2^-24 from rounding
    # its argument besides 1 ulp, and the silu takes four more operations
    err = 1.1 * ge * (np.abs(u) + ue) + (np.abs(s) + 1.1 * ge) * ue + (8 + np.abs(g)) * 2.0 ** -23 * np.abs(s * u)
    y = pkg.mxfp4_swiglu(x, w1, w3, out_dtype=torch.float32)
    assert (np.abs(_np(y) - s * u) <= err + 1e-37).all()
    t = pkg.quantize_mxfp4(x)
    out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=cuda)
    assert pkg.mxfp4_swiglu(t, w1, w3, out=out) is out and torch.equal(out, y.bfloat16())
    if N % 256 == 0:  # quantised in the epilogue: the blocks of the fp32 result
        q = pkg.mxfp4_swiglu(x, w1, w3, quantize=True)
        for a, b in zip(pkg.unpack_canonical(q), pkg.unpack_canonical(pkg.quantize_mxfp4(y))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("nmat,M,N,K", PLAN_SHAPES)
def test_every_planned_kernel(pkg, cuda, nmat, M, N, K):
    """Each kernel that a plan can choose, whole and in K pieces; the reference is a float64 product on
    the GPU of the dequantised operands (their quantisation is pinned above)."""
    print(f"case plan nmat={nmat} {M}x{N}x{K}", flush=True)
    dtype = DTYPES[(M + K) % 3]
    g = torch.Generator(device=cuda).manual_seed(N)
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    t = pkg.quantize_mxfp4(x)
    xd = pkg.dequantize(t).double()
    ws, refs, errs = [], [], []
    for _ in range(nmat):
        codes = torch.randint(0, 256, (N, K // 2), generator=g, device=cuda, dtype=torch.uint8)
        scales = torch.randint(116, 122, (N, K // 32), generator=g, device=cuda, dtype=torch.uint8)
        ws.append(pkg.pack_canonical(codes, scales, "mxfp4"))
        wd = pkg.dequantize(ws[-1]).double()
        refs.append(xd @ wd.T)
        errs.append(_sum_error(K, xd.abs() @ wd.abs().T))
        del wd
    if nmat == 1:
        ref, err = refs[0], errs[0]
        y = pkg.mxfp4_linear(x, ws[0], out_dtype=torch.float32)
        r = torch.randn(M, N, generator=g, device=cuda)
        z = pkg.mxfp4_linear(t, ws[0], residual=r)
        full = ref + r.double()
        assert ((z.double() - full).abs() <= err + 2.0 ** -8 * (full.abs() + err)).all()
        assert torch.equal(pkg.mxfp4_linear(t, ws[0], out_dtype=torch.float32), y)
    else:
        (gt, u), (ge, ue) = refs, errs
        s = gt * torch.sigmoid(gt)
        ref = s * u
        err = (1.1 * ge * (u.abs() + ue) + (s.abs() + 1.1 * ge) * ue + (8 + gt.abs()) * 2.0 ** -23 * ref.abs()) + 1e-37
        y = pkg.mxfp4_swiglu(x, *ws, out_dtype=torch.float32)
        if N % 256 == 0:
            q = pkg.mxfp4_swiglu(t, *ws, quantize=True)
            for a, b in zip(pkg.unpack_canonical(q), pkg.unpack_canonical(pkg.quantize_mxfp4(y))):
                assert torch.equal(a, b)
        assert torch.equal(pkg.mxfp4_swiglu(t, *ws), y.bfloat16())
    assert ((y.double() - ref).abs() <= err).all()


def test_rows_that_are_not_numbers_stay_in_their_row(pkg, cuda):
    for M in (3, 40, 200):
        x, xd, w, wd = _product_case(pkg, cuda, M, 512, 320, torch.float32)
        w3, _ = _weight(pkg, 512, 320, 5, cuda)
        clean = [pkg.mxfp4_linear(x, w, out_dtype=torch.float32), pkg.mxfp4_swiglu(x, w, w3, out_dtype=torch.float32)]
        x[1, 70], x[M - 1, 319] = float("inf"), float("nan")
        for y, ref in zip((pkg.mxfp4_linear(x, w, out_dtype=torch.float32),
                           pkg.mxfp4_swiglu(x, w, w3, out_dtype=torch.float32)), clean):
            for m in range(M):
                assert torch.isnan(y[m]).all() if m in (1, M - 1) else torch.equal(y[m], ref[m])
        d = pkg.dequantize(pkg.mxfp4_swiglu(x, w, w3, quantize=True))
        assert torch.isnan(d[1]).all() and torch.isnan(d[M - 1]).all() and torch.isfinite(d[0]).all()


@pytest.mark.parametrize("byte", [0, 1, 64, 127, 200, 225])
def test_scales_over_their_whole_range(pkg, cuda, byte):
    """Checkpoint scales down to the smallest.  |x| < 2^9 and a weight is at most 6 2^(byte - 127), so that
    no sum of 288 products reaches 2^(9 + 3 + 9 + byte - 127) < 2^127.  On top of the sums' rounding each
    product, and each of at most as many sums, may lose what is below the smallest normal number, 2^-126."""
    K, N = 288, 256
    codes = np.random.default_rng(byte).integers(0, 16, (N, K), dtype=np.uint8)
    scales = np.full((N, K // 32), byte, dtype=np.uint8)
    w = pkg.pack_canonical(torch.from_numpy(omx.join(codes)).to(cuda), torch.from_numpy(scales).to(cuda), "mxfp4")
    for M in (1, 5, 40, 300):
        print(f"case scale {byte} M={M}", flush=True)
        x = _rows(M, K, torch.float32, M).clamp(-256, 256)
        ref, mag = omx.linear(omx.dequantize(*omx.quantize(x.double().numpy())), omx.dequantize(codes, scales))
        y = pkg.mxfp4_linear(x.to(cuda), w, out_dtype=torch.float32)
        assert (np.abs(_np(y) - ref) <= _sum_error(K, mag) + 2 * K * 2.0 ** -126).all()


def test_offsets_beyond_32_bits(pkg, cuda):
    # rows 3.4 GB apart
    K, stride = 256, 1600 * 2 ** 20
    w, wd = _weight(pkg, 64, K, 3, cuda)
    wide = torch.empty(2 * stride + K, dtype=torch.bfloat16, device=cuda)
    x = wide.as_strided((3, K), (stride, 1))
    rows = _rows(3, K, torch.bfloat16, 1)
    x.copy_(rows.to(cuda))
    near = rows.to(cuda)
    for a, b in zip(pkg.unpack_canonical(pkg.quantize_mxfp4(x)), pkg.unpack_canonical(pkg.quantize_mxfp4(near))):
        assert torch.equal(a, b)
    assert torch.equal(pkg.mxfp4_linear(x, w), pkg.mxfp4_linear(near, w))
    norm = torch.zeros(K, dtype=torch.bfloat16, device=cuda)
    for a, b in zip(pkg.unpack_canonical(pkg.quantize_mxfp4(x, norm_weight=norm)),
                    pkg.unpack_canonical(pkg.quantize_mxfp4(near, norm_weight=norm))):
        assert torch.equal(a, b)
    del wide, x
    # an output of more than 2^31 values, and a product's largest number of tokens
    M, N, K = 65536, 33000, 32
    w, wd = _weight(pkg, N, K, 4, cuda)
    some = torch.randn(64, K, generator=torch.Generator().manual_seed(5)).bfloat16()
    y = pkg.mxfp4_linear(some.to(cuda).repeat(M // 64, 1), w)
    ref, mag = omx.linear(omx.dequantize(*omx.quantize(some.double().numpy())), wd)
    first = y[:64]
    assert (np.abs(_np(first) - ref) <= _bf16_error(ref, _sum_error(K, mag))).all()
    for r in (64, 32768, M - 64):
        assert torch.equal(y[r:r + 64], first)


def test_guarded_outputs(pkg, cuda):
    """Nothing is written outside the output, whatever the tail sizes."""
    for M, N, K in ((1, 33, 64), (5, 3, 256), (33, 250, 512), (70, 515, 288), (200, 129, 544)):
        x, _, w, _ = _product_case(pkg, cuda, M, N, K, torch.bfloat16)
        w3, _ = _weight(pkg, N, K, 8, cuda)
        for dt in (torch.bfloat16, torch.float32):
            for f in (lambda o: pkg.mxfp4_linear(x, w, out=o), lambda o: pkg.mxfp4_swiglu(x, w, w3, out=o)):
                flat = torch.full((M * N + 4096,), 3.0, dtype=dt, device=cuda)
                o = flat[2048:2048 + M * N].view(M, N)
                f(o)
                assert (flat[:2048] == 3.0).all() and (flat[2048 + M * N:] == 3.0).all()


def test_misfits_are_refused(pkg, cuda):
    x, _, w, _ = _product_case(pkg, cuda, 4, 64, 256, torch.bfloat16)
    t = pkg.quantize_mxfp4(x)
    bad = [dict(out=torch.empty(4, 65, device=cuda)), dict(out=torch.empty(4, 64, device=cuda, dtype=torch.float16)),
           dict(out=torch.empty(64, 4, device=cuda).T), dict(residual=torch.empty(4, 32, device=cuda)),
           dict(residual=torch.empty(4, 64, device=cuda, dtype=torch.float16)), dict(residual=torch.empty(4, 64)),
           dict(out=torch.empty(4, 64, device=cuda), out_dtype=torch.bfloat16),
           dict(out=torch.empty(4 * 64 + 1, device=cuda)[1:].view(4, 64))]
    for kw in bad:
        with pytest.raises(ValueError):
            pkg.mxfp4_linear(t, w, **kw)
    with pytest.raises(ValueError):
        pkg.mxfp4_linear(x[:, :128], w)
    with pytest.raises(ValueError, match="columns"):
        pkg.mxfp4_linear(t, pkg.pack_weight(torch.ones(64, 288, dtype=torch.bfloat16, device=cuda), "mxfp4"))
    narrow = pkg.pack_weight(torch.ones(32, 256, dtype=torch.bfloat16, device=cuda), "mxfp4")
    with pytest.raises(ValueError, match="rows"):
        pkg.mxfp4_swiglu(t, w, narrow)
    with pytest.raises(ValueError, match="256"):
        pkg.mxfp4_swiglu(t, w, w, quantize=True)
    with pytest.raises(ValueError, match="quantize"):
        pkg.mxfp4_swiglu(t, w, w, quantize=True, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="out_dtype"):
        pkg.mxfp4_linear(t, w, out_dtype=torch.float16)
    for short in (pkg.MxTensor(t.buf, 33, 256), pkg.MxTensor(t.buf[16:], 4, 256), pkg.MxTensor(t.buf.view(torch.int8), 4, 256),
                  pkg.MxTensor(t.buf, 0, 256), pkg.MxTensor(t.buf, 4, 48)):  # a buffer that is not the shape's
        for f in (pkg.dequantize, pkg.unpack_canonical, lambda v: pkg.mxfp4_linear(v, w)):
            with pytest.raises(ValueError):
                f(short)
    with pytest.raises(ValueError):
        pkg.mxfp4_linear(t, pkg.PackedWeight(w.buf, 65, 256, "mxfp4"))
    r = torch.zeros(4, 64, device=cuda)
    with pytest.raises(ValueError):  # in place of another dtype
        pkg.mxfp4_linear(t, w, residual=r, out=r.view(torch.bfloat16)[:, :64])


# ---------------------------------------------------------------- streams, graphs


@pytest.mark.parametrize("M", [1, 40, 300])
def test_graph_replays(pkg, cuda, M):
    N, K = 512, 1056
    x, _, w, _ = _product_case(pkg, cuda, M, N, K, torch.bfloat16)
    w3, _ = _weight(pkg, N, K, 4, cuda)
    wd, _ = _weight(pkg, 320, N, 6, cuda)

    def chain(v):
        h = pkg.mxfp4_swiglu(v, w, w3, quantize=True)
        return pkg.mxfp4_linear(h, wd, out_dtype=torch.float32)

    static = x.clone()
    for _ in range(2):
        chain(static)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of one process share no scratch that a replay of the other needs
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = chain(static)
        graphs.append((g, y))
    for i in range(4):
        new = _rows(M, K, torch.bfloat16, 50 + i).to(cuda)
        eager = chain(new)
        static.copy_(new)
        for g, y in graphs:
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
            torch.empty(1 << 20, device=cuda).fill_(1.0)


def test_two_streams_at_once(pkg, cuda):
    N, K = 2048, 2048
    cases = [_product_case(pkg, cuda, M, N, K, torch.bfloat16, seed=M) for M in (3, 100)]
    want = [pkg.mxfp4_linear(x, w, out_dtype=torch.float32) for x, _, w, _ in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, (x, _, w, _)) in enumerate(zip(streams, cases)):
            if len(got[i]) % 2:
                with torch.cuda.stream(s):
                    got[i].append(pkg.mxfp4_linear(x, w, out_dtype=torch.float32))
            else:
                got[i].append(pkg.mxfp4_linear(x, w, out_dtype=torch.float32, stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


# ---------------------------------------------------------------- the block


def _state_dict(H, I, cuda, seed=1):
    g = torch.Generator().manual_seed(seed)
    shapes = {"gate_proj.weight": (I, H), "up_proj.weight": (I, H), "down_proj.weight": (H, I)}
    return {k: (torch.randn(*s, generator=g) * 0.05).bfloat16().to(cuda) for k, s in shapes.items()}


@pytest.mark.parametrize("H,I,M", [(256, 512, 1), (256, 512, 7), (1024, 2304, 16), (512, 256, 33), (768, 1280, 130),
                                   (512, 1024, 300), (1280, 512, 700)])
def test_block(pkg, cuda, H, I, M):
    """The block is its pieces one after the other, and its down projection is the oracle's product of the
    h that the gate/up pair left."""
    print(f"case block H={H} I={I} M={M}", flush=True)
    mlp = pkg.Qwen36MLP(cuda, _state_dict(H, I, cuda), weight_format="mxfp4", max_tokens=M)
    w = mlp.weights
    assert mlp.weight_format == "mxfp4" and w.w2.fmt == "mxfp4"
    x = _rows(M, H, torch.bfloat16, 3, 0.05).to(cuda)
    r = torch.randn(M, H, generator=torch.Generator().manual_seed(4)).to(cuda)
    h = pkg.mxfp4_swiglu(pkg.quantize_mxfp4(x), w.w1, w.w3, quantize=True)
    y = mlp.forward(x.view(1, 1, M, H), residual=r.view(1, 1, M, H), out_dtype=torch.float32).view(M, H)
    assert torch.equal(y, pkg.mxfp4_linear(h, w.w2, residual=r, out_dtype=torch.float32))
    ref, mag = omx.linear(_np(pkg.dequantize(h)), _np(pkg.dequantize(w.w2)))
    ref, err = ref + _np(r), _sum_error(I, mag)
    assert (np.abs(_np(y) - ref) <= err + 2.0 ** -24 * (np.abs(ref) + err)).all()
    assert torch.equal(mlp.forward(x, residual=r), y.bfloat16())
    plain = mlp.forward(x)
    assert torch.equal(plain, pkg.mxfp4_linear(h, w.w2))
    # the library's own scratch
    if M <= 32:
        from qwen_mlp_amd import _lib

        out = torch.empty_like(x)
        _lib.check(_lib.lib().qmlp_forward_noalloc(_lib.ptr(x), _lib.ptr(w.w1.buf), _lib.ptr(w.w3.buf),
                                                   _lib.ptr(w.w2.buf), None, _lib.ptr(out), M, H, I, _lib.FMT_MXFP4, 0,
                                                   _lib.stream_handle()), "qmlp_forward_noalloc")
        assert torch.equal(out, plain)
    # the norm in front, in place
    nw = (torch.randn(H, generator=torch.Generator().manual_seed(5)) * 0.1).bfloat16().to(cuda)
    hn = pkg.mxfp4_swiglu(pkg.quantize_mxfp4(x, norm_weight=nw), w.w1, w.w3, quantize=True)
    want = pkg.mxfp4_linear(hn, w.w2, residual=x)
    assert torch.equal(mlp.forward_rmsnorm(x, nw), want)
    z = x.clone()
    assert torch.equal(mlp.forward_rmsnorm(z, nw, out=z), want)


def test_pool_shared_with_other_formats(pkg, cuda):
    """A workspace that MXFP4 forwards used serves the formats that count arrivals in it, and back."""
    H, I, M = 512, 1024, 16
    sd = _state_dict(H, I, cuda)
    pool = pkg.WorkspacePool()
    mlps = [pkg.Qwen36MLP(cuda, sd, weight_format=f, max_tokens=300, pool=pool) for f in ("bfp8", "mxfp4", "bf16")]
    x = _rows(M, H, torch.bfloat16, 3, 0.05).to(cuda)
    big = _rows(300, H, torch.bfloat16, 4, 0.05).to(cuda)
    first = [m.forward(x) for m in mlps]
    for _ in range(3):
        for m, f in zip(mlps, first):
            m.forward(big)
            assert torch.equal(m.forward(x), f)


def test_load_cache_and_packer(pkg, cuda, tmp_path):
    from safetensors.torch import save_file

    from qwen_mlp_amd import pack_checkpoint

    H, I = 256, 512
    sd = _state_dict(H, I, cuda)
    a = pkg.load_mlp_weights(cuda, sd, tmp_path / "cache", weight_format="mxfp4")
    b = pkg.load_mlp_weights(cuda, {}, tmp_path / "cache", weight_format="mxfp4")
    save_file({f"model.layers.0.mlp.{k}": v.cpu() for k, v in sd.items()}, str(tmp_path / "model.safetensors"))
    assert pack_checkpoint.main(["--checkpoint", str(tmp_path), "--out", str(tmp_path / "out"), "--format", "mxfp4",
                                 "--planar"]) == 0
    c = pkg.load_mlp_weights(cuda, {}, tmp_path / "out" / "layer_0", weight_format="mxfp4")
    for name in ("w1", "w2", "w3"):
        for other in (b, c):
            assert torch.equal(getattr(a, name).buf, getattr(other, name).buf)
    q, e = np.load(tmp_path / "out" / "layer_0" / "up_proj.q.npy"), np.load(tmp_path / "out" / "layer_0" / "up_proj.e8.npy")
    want, wants = omx.quantize(_np(sd["up_proj.weight"]))
    assert np.array_equal(q, omx.join(want)) and np.array_equal(e, wants)


def _head(pkg, t, rows):
    """The first ``rows`` rows (a multiple of 32) of a packed matrix."""
    return pkg.MxTensor(t.buf[:omx.packed_bytes(rows, t.cols)], rows, t.cols)


def test_block_beyond_32_bit_offsets(pkg, cuda):
    """The block at its largest number of tokens, with more than 2^30 values of h: its pieces, the same in
    every copy of the tokens, and right in the first."""
    H, I, M, rows = 256, 16640, 65536, 64
    mlp = pkg.Qwen36MLP(cuda, _state_dict(H, I, cuda), weight_format="mxfp4", max_tokens=64, pool=pkg.WorkspacePool())
    w = mlp.weights
    some = _rows(rows, H, torch.bfloat16, 3, 0.05).to(cuda)
    x = some.repeat(M // rows, 1)
    r = torch.randn(M, H, generator=torch.Generator(device=cuda).manual_seed(4), device=cuda)
    h = pkg.mxfp4_swiglu(x, w.w1, w.w3, quantize=True)
    y = mlp.forward(x, residual=r, out_dtype=torch.float32)
    assert torch.equal(y, pkg.mxfp4_linear(h, w.w2, residual=r, out_dtype=torch.float32))
    plain = mlp.forward(x)
    for at in (rows, M // 2, M - rows):
        assert torch.equal(plain[at:at + rows], plain[:rows])
    # h of the first copy: half a step of a value of its block (at most the scale itself), a block's
    # largest values saturate by at most twice the scale, and the sums' rounding
    (codes, scales), xd = _unpack(pkg, _head(pkg, h, rows)), omx.dequantize(*omx.quantize(_np(some)))
    hd = omx.dequantize(codes, scales)
    (g, gm), (u, um) = (omx.linear(xd, _np(pkg.dequantize(v))) for v in (w.w1, w.w3))
    ge, ue, s = _sum_error(H, gm), _sum_error(H, um), _silu(g)
    err = 1.1 * ge * (np.abs(u) + ue) + (np.abs(s) + 1.1 * ge) * ue + (8 + np.abs(g)) * 2.0 ** -23 * np.abs(s * u)
    step = np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, axis=1)
    assert (np.abs(hd - s * u) <= 2 * step + err).all()
    ref, mag = omx.linear(hd, _np(pkg.dequantize(w.w2)))
    ref, err = ref + _np(r[:rows]), _sum_error(I, mag)
    assert (np.abs(_np(y[:rows]) - ref) <= err + 2.0 ** -24 * (np.abs(ref) + err)).all()
    # the norm in front
    nw = (torch.randn(H, generator=torch.Generator().manual_seed(5)) * 0.1).bfloat16().to(cuda)
    hn = pkg.mxfp4_swiglu(pkg.quantize_mxfp4(x, norm_weight=nw), w.w1, w.w3, quantize=True)
    assert torch.equal(mlp.forward_rmsnorm(x, nw), pkg.mxfp4_linear(hn, w.w2, residual=x))


def test_largest_scales(pkg, cuda):
    """Scales of 252 to 254: magnitudes from 2^128 on, no fp32 or bf16 numbers, dequantise to infinities, the
    others exactly.  In a product with small activations they count as what they are: |x| < 2^-90, so that
    no sum of 288 products reaches 2^(9 + 3 + 127 - 90) = 2^49."""
    K, N = 288, 96
    codes = np.random.default_rng(1).integers(0, 16, (N, K), dtype=np.uint8)
    codes[:, :16] = np.arange(16)
    scales = np.tile(np.array([252, 253, 254], dtype=np.uint8), (N, 3))
    w = pkg.pack_canonical(torch.from_numpy(omx.join(codes)).to(cuda), torch.from_numpy(scales).to(cuda), "mxfp4")
    wd = omx.dequantize(codes, scales)
    big = np.abs(wd) >= 2.0 ** 128
    assert big.any() and (np.abs(wd[~big]) > 2.0 ** 127).any()
    for dt in (torch.float32, torch.bfloat16):
        d = _np(pkg.dequantize(w, dtype=dt))
        assert np.array_equal(d[~big], wd[~big]) and np.array_equal(d[big], np.sign(wd[big]) * np.inf)
    for M in (1, 5, 40):
        x = (_rows(M, K, torch.float32, M).clamp(-256, 256) * 2.0 ** -98).contiguous()
        ref, mag = omx.linear(omx.dequantize(*omx.quantize(x.double().numpy())), wd)
        y = pkg.mxfp4_linear(x.to(cuda), w, out_dtype=torch.float32)
        assert (np.abs(_np(y) - ref) <= _sum_error(K, mag)).all()


# ---------------------------------------------------------------- largest sizes, streams, checkpoints


@pytest.mark.parametrize("rows,cols", [(1 << 20, 32), (2, 1 << 20)])
def test_largest_matrices(pkg, cuda, rows, cols):
    """As activations and as weights, against the oracle on some of their rows and against each other."""
    print(f"case largest {rows}x{cols}", flush=True)
    base = _rows(min(rows, 96), cols, torch.bfloat16, 9)
    x = base.to(cuda).repeat(-(-rows // 96), 1)[:rows].contiguous()
    t = pkg.quantize_mxfp4(x)
    codes, scales = pkg.unpack_canonical(t)
    want, wants = omx.quantize(_np(base))
    assert np.array_equal(codes[:96].cpu().numpy(), omx.join(want)) and np.array_equal(scales[:96].cpu().numpy(), wants)
    for at in (range(96, rows - 95, 96 * 1021) if rows > 96 else ()):
        assert torch.equal(codes[at:at + 96], codes[:96]) and torch.equal(scales[at:at + 96], scales[:96])
    assert torch.equal(codes[-1], codes[(rows - 1) % 96]) and torch.equal(scales[-1], scales[(rows - 1) % 96])
    pw = pkg.pack_weight(x, "mxfp4")
    units = t.nbytes - omx.TRAILER_BYTES  # rows is whole units here, or the rest is zeros in a weight
    if rows % 32 == 0:
        assert torch.equal(pw.buf[:units], t.buf[:units])
    again = pkg.pack_canonical(codes, scales, "mxfp4")
    assert torch.equal(again.buf, pw.buf)
    assert torch.equal(pkg.dequantize(pw, dtype=torch.bfloat16), pkg.dequantize(t, dtype=torch.bfloat16))
    normed = pkg.quantize_mxfp4(x, norm_weight=torch.zeros(cols, dtype=torch.bfloat16, device=cuda))
    few = pkg.quantize_mxfp4(x[:96], norm_weight=torch.zeros(cols, dtype=torch.bfloat16, device=cuda))
    for a, b in zip(pkg.unpack_canonical(normed), pkg.unpack_canonical(few)):
        assert torch.equal(a[:96], b) and torch.equal(a[-1], b[(rows - 1) % 96])


@pytest.mark.parametrize("M,N,K", [(1, 1 << 20, 64), (70, 1 << 20, 64), (1, 33, 1 << 20), (40, 33, 1 << 20),
                                   (1100, 33, 1 << 20)])
def test_products_at_the_largest_sizes(pkg, cuda, M, N, K):
    """Every block's scale is the same, so every product is a multiple of 2^-9.  A random sum of 2^20 of them, up
    to 36 2^-7 = 144 units each, stays below 2^24 units (it has a spread of 2^10 times 40 or so), so that no
    sum rounds.  For a gate below -87.33 the reciprocal of 1 + exp(-gate) lies below fp32's
    normal numbers, and the silu may come out as 0, from which it is less than 87.34 e^-87.33 < 1.1e-36 away."""
    print(f"case largest product {M}x{N}x{K}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(N)
    table = torch.tensor([*omx.VALUES, *-omx.VALUES], dtype=torch.float32, device=cuda)
    x = table[torch.randint(0, 16, (M, K), generator=g, device=cuda)]
    x[:, ::32] = 4.0
    t = pkg.quantize_mxfp4(x)
    assert torch.equal(pkg.dequantize(t), x)
    scales = torch.full((N, K // 32), 120, device=cuda, dtype=torch.uint8)
    ws = [pkg.pack_canonical(torch.randint(0, 256, (N, K // 2), generator=g, device=cuda, dtype=torch.uint8), scales,
                             "mxfp4") for _ in range(2)]
    some = [0, M // 2, M - 1]
    gate, up = (x[some].double() @ pkg.dequantize(w).double().T for w in ws)
    y = pkg.mxfp4_linear(x, ws[0], out_dtype=torch.float32)
    assert torch.equal(y[some].double(), gate)
    assert torch.equal(pkg.mxfp4_linear(t, ws[0], out_dtype=torch.float32), y)
    ref = gate * torch.sigmoid(gate) * up
    y = pkg.mxfp4_swiglu(x, *ws, out_dtype=torch.float32)
    err = (8 + gate.abs()) * 2.0 ** -23 * ref.abs() + 1.1e-36 * up.abs() + 1e-37
    assert ((y[some].double() - ref).abs() <= err).all()
    assert torch.equal(pkg.mxfp4_swiglu(t, *ws), y.bfloat16())


def test_every_call_on_a_given_stream(pkg, cuda):
    """``stream`` may be another one than the current one; what it returns is ready on that stream."""
    x, _, w, _ = _product_case(pkg, cuda, 40, 512, 320, torch.bfloat16)
    w3, _ = _weight(pkg, 512, 320, 5, cuda)
    plain = torch.randn(512, 256, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda)
    norm = torch.zeros(320, dtype=torch.bfloat16, device=cuda)
    q, e = pkg.unpack_canonical(w)
    t = pkg.quantize_mxfp4(x)
    calls = [lambda **k: pkg.quantize_mxfp4(x, **k).buf[:64], lambda **k: pkg.quantize_mxfp4(x, norm_weight=norm, **k).buf[:64],
             lambda **k: pkg.dequantize(w, **k), lambda **k: pkg.dequantize(t, dtype=torch.bfloat16, **k),
             lambda **k: pkg.unpack_canonical(t, **k)[0], lambda **k: pkg.pack_canonical(q, e, "mxfp4", **k).buf,
             lambda **k: pkg.mxfp4_linear(x, w, **k), lambda **k: pkg.mxfp4_swiglu(x, w, w3, **k),
             lambda **k: pkg.dequantize(pkg.mxfp4_swiglu(x, w, w3, quantize=True, **k), **k)]
    calls += [lambda f=f, **k: pkg.pack_weight(plain, f, **k).buf for f in ("mxfp4", "bfp8", "bf4", "bf16")]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for f, y in zip(calls, want):
        got = f(stream=s)
        s.synchronize()
        assert torch.equal(got, y)
    assert torch.cuda.current_stream() != s


def test_a_block_from_a_checkpoint_in_the_format(pkg, cuda, tmp_path):
    """Codes and scales become a block through MLPWeights, or a Qwen36MLP through the weight cache, and mean
    the values that they stand for."""
    from qwen_mlp_amd import weight_cache

    H, I, M = 256, 512, 7
    rng = np.random.default_rng(3)
    made, values = {}, {}
    for name, (rows, cols) in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I))):
        codes = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
        scales = rng.integers(117, 124, (rows, cols // 32), dtype=np.uint8)
        made[name] = pkg.pack_canonical(torch.from_numpy(omx.join(codes)).to(cuda), torch.from_numpy(scales).to(cuda), "mxfp4")
        values[name] = omx.dequantize(codes, scales)
        weight_cache.save(weight_cache.cache_file(tmp_path, name, "mxfp4"), made[name])
    weights = pkg.MLPWeights(w1=made["gate_proj"], w2=made["down_proj"], w3=made["up_proj"])
    x = _rows(M, H, torch.bfloat16, 3, 0.05).to(cuda)
    y = pkg.mlp_forward(x, weights, residual=x, out_dtype=torch.float32)
    mlp = pkg.Qwen36MLP(cuda, {}, tmp_path, weight_format="mxfp4", max_tokens=M)
    assert torch.equal(mlp.forward(x, residual=x, out_dtype=torch.float32), y)
    h = pkg.mxfp4_swiglu(x, made["gate_proj"], made["up_proj"], quantize=True)
    ref, mag = omx.linear(_np(pkg.dequantize(h)), values["down_proj"])
    ref, err = ref + _np(x), _sum_error(I, mag)
    assert (np.abs(_np(y) - ref) <= err + 2.0 ** -24 * (np.abs(ref) + err)).all()


def test_verify_arm_on_the_format(pkg, cuda):
    """The arm's check of each layer's weights and its route take mxfp4 layers."""
    from qwen_mlp_amd.verify_arm import VerifyArm

    H, I = 256, 512

    class Decoder:
        def __init__(self, seed):
            self.sd = _state_dict(H, I, cuda, seed)

        def state_dict(self):
            return self.sd

        def forward(self, x):
            return None

    layers = [Decoder(1), Decoder(2)]
    amd = [pkg.Qwen36MLP(cuda, d.sd, weight_format="mxfp4", max_tokens=16) for d in layers]
    x = _rows(16, H, torch.bfloat16, 3, 0.05).to(cuda).view(1, 1, 16, H)
    arm = VerifyArm(layers, amd)
    with arm.install():
        got = [d.forward(x) for d in layers]
    assert all(torch.equal(y, m.forward(x)) for y, m in zip(got, amd)) and arm.audit["hits"] == [1, 1]
    with pytest.raises(ValueError, match="layer 0"):
        VerifyArm(layers, amd[::-1]).check_layer_weights()
