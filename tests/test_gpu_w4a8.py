"""8-bit activations with 4-bit weights on the GPU against the oracles' definitions in 64 bits.

Quantisation, its layout and dequantisation are compared bit for bit.  A product's operands are integers
(7 bits and a sign) times powers of two and 4-bit values, each multiplied as two digits of one sign, so every
single product is exact and only the fp32 sums round: the matrix cores take K in steps of 64 and each step as
two products, each of which rounds at most twice (its own sum of 64 terms, then the accumulator) by at most
2^-23 of the magnitudes summed so far; splitting K over waves or pieces adds at most 32 more additions.
``_sum_error`` is that bound; an output's own rounding to bf16 comes on top (half a step, 2^-8 of the value)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mxfp4 as omx
from oracle import mxint8 as omi
from test_w4a8 import PLAN_SHAPES

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _sum_error(K, magnitudes):
    return (4 * (K / 64 + 1) + 32) * 2.0 ** -23 * magnitudes


def _bf16_error(y, err):
    return err + 2.0 ** -8 * (np.abs(y) + err)


def _np(t):
    return t.double().cpu().numpy()


def _rows(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * scale
    x *= torch.exp2(torch.randint(-6, 7, (rows, cols // 32, 1), generator=g).float()).expand(-1, -1, 32).reshape(rows, cols)
    return x.to(dtype)


def _weight(pkg, rows, cols, seed, device):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    scales = rng.integers(117, 125, (rows, cols // 32), dtype=np.uint8)
    pw = pkg.pack_canonical(torch.from_numpy(omx.join(codes)).to(device), torch.from_numpy(scales).to(device), "mxfp4")
    return pw, omx.dequantize(codes, scales)


def _unpack(pkg, t):
    q, e = pkg.unpack_canonical(t)
    return q.cpu().numpy(), e.cpu().numpy()


# ---------------------------------------------------------------- the format


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 5120), (3, 64), (8, 256), (17, 288), (33, 224), (257, 1056),
                                       (1030, 8320)])
def test_quantize_is_the_definition(pkg, cuda, rows, cols, dtype):
    print(f"case quantize {rows}x{cols} {dtype}", flush=True)
    x = _rows(rows, cols, dtype, rows + cols)
    t = pkg.quantize_mxint8(x.to(cuda))
    assert t.shape == (rows, cols) and t.buf.numel() == omi.packed_bytes(rows, cols)
    q, scales = _unpack(pkg, t)
    want, wants = omi.quantize(x.double().numpy())
    assert np.array_equal(scales, wants) and np.array_equal(q, want)
    if rows * cols < 10000:
        buf = t.buf.cpu().numpy()
        for at, b in omi.packed_rows(want, wants, np.signbit(x.double().numpy())):
            assert np.array_equal(buf[at:at + len(b)], b), at
    d = omi.dequantize(want, wants)
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
    t = pkg.quantize_mxint8(x.to(cuda))
    q, scales = _unpack(pkg, t)
    want, wants = omi.quantize(x.double().numpy())
    assert np.array_equal(scales, wants) and np.array_equal(q, want)
    assert np.array_equal(_np(pkg.dequantize(t, dtype=torch.bfloat16)), omi.dequantize(want, wants), equal_nan=True)


def test_quantize_strided_rows(pkg, cuda):
    for dtype, pad in ((torch.bfloat16, 8), (torch.float32, 4), (torch.float16, 40)):
        wide = _rows(21, 160, dtype, 3).to(cuda)
        wide = torch.cat([wide, torch.full((21, pad), float("nan"), dtype=dtype, device=cuda)], dim=1)
        x = wide[:, :160]
        assert not x.is_contiguous()
        a, b = pkg.quantize_mxint8(x), pkg.quantize_mxint8(x.contiguous())
        for u, v in zip(pkg.unpack_canonical(a), pkg.unpack_canonical(b)):
            assert torch.equal(u, v)
    for bad in (wide[:, 1:161], wide.T, wide[:, :160:2], wide[:, :16], wide[:0, :160], wide[0], wide.to(torch.float64)):
        with pytest.raises(ValueError):
            pkg.quantize_mxint8(bad)


# ---------------------------------------------------------------- the norm

NORM_SHAPES = [(1, 32), (1, 5120), (3, 96), (16, 5120), (5, 288), (33, 1056), (300, 512), (2, 17408), (40, 8192),
               (130, 5120), (1000, 2080), (2, 33024)]


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("xt,rt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                   (torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                   (torch.bfloat16, None), (torch.float32, None)])
def test_add_rmsnorm(pkg, cuda, rows, cols, xt, rt):
    """h is the rounded sum, bit for bit (one fp32 addition of two values of at most 24 bits, rounded to fp32,
    then to bf16: both roundings are the same in the oracle).  n: the norm's fp32 error (a sum of squares of
    non-negative terms in at most cols / 512 + 30 steps and a few operations, below 2^-17 of the value)
    moves n by one bf16 step where a rounding border lies that near, and only there.  The packed matrix is the
    quantisation of the rows, bit for bit."""
    print(f"case add_rmsnorm {rows}x{cols} {xt} {rt}", flush=True)
    x = _rows(rows, cols, xt, 11)
    r = None if rt is None else _rows(rows, cols, rt, 12, 2.0)
    w = (torch.randn(cols, generator=torch.Generator().manual_seed(2)) * 0.1).bfloat16()
    r_gpu = None if r is None else r.to(cuda)
    h, n, q = pkg.add_rmsnorm(x.to(cuda), r_gpu, w.to(cuda), eps=1e-5, output="both")
    want_h = x if r is None else (x.float() + r.float()).to(rt)
    assert torch.equal(h.cpu(), want_h) and h.dtype == want_h.dtype
    d = want_h.double()
    exact = d / torch.sqrt((d * d).mean(dim=1, keepdim=True) + 1e-5) * (1 + w.double())
    lo, hi = (exact * (1 - 2.0 ** -17)).bfloat16(), (exact * (1 + 2.0 ** -17)).bfloat16()
    got = n.cpu()
    assert ((got == lo) | (got == hi)).all()
    assert (got == exact.bfloat16()).float().mean() > 0.97
    for a, b in zip(pkg.unpack_canonical(q), pkg.unpack_canonical(pkg.quantize_mxint8(n))):
        assert torch.equal(a, b)
    buf = q.buf.cpu().numpy()
    if rows * cols < 10000:  # the padding up to the unit's end
        for at, b in omi.packed_rows(*_unpack(pkg, q), np.signbit(_np(n))):
            assert np.array_equal(buf[at:at + len(b)], b), at
    # one output alone, given and in-place sums, strided rows: the same bits
    h2, n2 = pkg.add_rmsnorm(x.to(cuda), r_gpu, w.to(cuda), eps=1e-5, output="rows")
    h3, q3 = pkg.add_rmsnorm(x.to(cuda), r_gpu, w.to(cuda), eps=1e-5)
    assert torch.equal(n2, n) and torch.equal(h2, h) and torch.equal(h3, h)
    for a, b in zip(pkg.unpack_canonical(q), pkg.unpack_canonical(q3)):
        assert torch.equal(a, b)
    wide = torch.cat([x, x], dim=1).to(cuda)[:, :cols]
    if r is not None:
        inplace = torch.cat([r, r], dim=1).to(cuda)
        h4, n4 = pkg.add_rmsnorm(wide, inplace[:, :cols], w.to(cuda), eps=1e-5, output="rows", out=inplace[:, :cols])
        assert torch.equal(h4, h) and torch.equal(n4, n)
        assert torch.equal(inplace[:, cols:].cpu(), r)
        given = torch.zeros(rows, cols, dtype=rt, device=cuda)
        assert pkg.add_rmsnorm(wide, r_gpu, w.to(cuda), eps=1e-5, out=given)[0] is given and torch.equal(given, h)
    else:
        assert torch.equal(pkg.add_rmsnorm(wide, None, w.to(cuda), eps=1e-5, output="rows")[1], n)


def test_add_rmsnorm_rows_that_are_not_numbers(pkg, cuda):
    x = _rows(4, 64, torch.float32, 1)
    x[1, 3], x[2, 40] = float("inf"), float("nan")
    w = torch.zeros(64, dtype=torch.bfloat16, device=cuda)
    h, n, q = pkg.add_rmsnorm(x.to(cuda), torch.zeros(4, 64, device=cuda), w, output="both")
    assert torch.equal(h.cpu(), x) or torch.allclose(h.cpu(), x, equal_nan=True)
    assert n[2].isnan().all() and not n[[0, 3]].isnan().any()
    v = pkg.dequantize(q)
    assert v[2].isnan().all() and not v[[0, 3]].isnan().any()
    assert v[1, :32].isnan().all()  # inf / inf; the other block's values over an infinite norm are zeros
    assert (v[1, 32:] == 0).all()
    zero, _, qz = pkg.add_rmsnorm(torch.zeros(2, 96, device=cuda), torch.zeros(2, 96, device=cuda),
                                  torch.ones(96, dtype=torch.bfloat16, device=cuda), output="both")
    assert (zero == 0).all() and (pkg.dequantize(qz) == 0).all()


# ---------------------------------------------------------------- the products

SHAPES = [(1, 1, 32), (1, 33, 64), (2, 100, 224), (5, 3, 1056), (16, 256, 288), (31, 31, 512), (32, 32, 256),
          (33, 64, 2080), (64, 1000, 96), (65, 130, 544), (100, 257, 1024), (128, 96, 4352), (257, 513, 800),
          (300, 1024, 256), (1, 5120, 5120), (4, 640, 4352), (1, 640, 17408), (17, 384, 8704), (513, 260, 2304),
          (1000, 300, 512)]


def _product_case(pkg, cuda, M, N, K, dtype, seed=0):
    x = _rows(M, K, dtype, M * 7 + K + seed)
    w, wd = _weight(pkg, N, K, N + K + seed, cuda)
    return x.to(cuda), omi.dequantize(*omi.quantize(x.double().numpy())), w, wd


def _linear_case(pkg, cuda, M, N, K, dtype):
    x, xd, w, wd = _product_case(pkg, cuda, M, N, K, dtype)
    ref, mag = omx.linear(xd, wd)
    err = _sum_error(K, mag)
    y = pkg.w4a8_linear(x, w, out_dtype=torch.float32)
    assert y.shape == (M, N) and y.dtype == torch.float32
    assert (np.abs(_np(y) - ref) <= err).all()
    t = pkg.quantize_mxint8(x)
    out = torch.full((M, N), 7.0, device=cuda)
    assert pkg.w4a8_linear(t, w, out=out) is out and torch.equal(out, y)
    yb = pkg.w4a8_linear(t, w)
    assert yb.dtype == torch.bfloat16 and torch.equal(yb, y.bfloat16())
    r = torch.randn(M, N, generator=torch.Generator().manual_seed(M)).to(cuda)
    y2 = pkg.w4a8_linear(t, w, residual=r, out_dtype=torch.float32)
    full = ref + _np(r)
    assert (np.abs(_np(y2) - full) <= err + 2.0 ** -24 * (np.abs(full) + err)).all()
    rb = r.bfloat16()
    y3 = pkg.w4a8_linear(x, w, residual=rb)
    full = ref + _np(rb)
    assert (np.abs(_np(y3) - full) <= _bf16_error(full, err * (1 + 2.0 ** -23))).all()
    inplace = rb.clone()
    assert torch.equal(pkg.w4a8_linear(x, w, residual=inplace, out=inplace), y3)
    assert torch.equal(pkg.w4a8_linear(t, w, residual=r, out=r), y2)


def _silu(g):
    return g / (1 + np.exp(-np.clip(g, -700, 700)))


def _swiglu_case(pkg, cuda, M, N, K, dtype):
    x, xd, w1, w1d = _product_case(pkg, cuda, M, N, K, dtype)
    w3, w3d = _weight(pkg, N, K, 99, cuda)
    g, gm = omx.linear(xd, w1d)
    u, um = omx.linear(xd, w3d)
    t = pkg.quantize_mxint8(x)
    gen = torch.Generator().manual_seed(N)
    add = [torch.randn(M, N, generator=gen).to(cuda) for _ in range(2)]
    for adds in ((None, None), (add[0], add[1]), (None, add[1]), (add[0], None)):
        gg, uu = (a if b is None else a + _np(b) for a, b in zip((g, u), adds))
        ge, ue = (_sum_error(K, m) + (0 if b is None else 2.0 ** -23 * (np.abs(a) + _sum_error(K, m)))
                  for m, a, b in zip((gm, um), (gg, uu), adds))
        s = _silu(gg)
        # |silu'| < 1.1; the kernel's exponential has a relative error of about |g| 2^-24 from rounding
        # its argument besides 1 ulp, and the silu takes four more operations
        err = (1.1 * ge * (np.abs(uu) + ue) + (np.abs(s) + 1.1 * ge) * ue
               + (8 + np.abs(gg)) * 2.0 ** -23 * np.abs(s * uu))
        y = pkg.w4a8_swiglu(x, w1, w3, gate_add=adds[0], up_add=adds[1], out_dtype=torch.float32)
        assert (np.abs(_np(y) - s * uu) <= err + 1e-37).all()
        out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=cuda)
        assert pkg.w4a8_swiglu(t, w1, w3, *adds, out=out) is out and torch.equal(out, y.bfloat16())
        if N % 256 == 0:  # quantised in the epilogue: the blocks of the fp32 result
            q = pkg.w4a8_swiglu(x, w1, w3, *adds, quantize=True)
            for a, b in zip(pkg.unpack_canonical(q), pkg.unpack_canonical(pkg.quantize_mxint8(y))):
                assert torch.equal(a, b)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(pkg, cuda, M, N, K):
    print(f"case linear {M}x{N}x{K}", flush=True)
    _linear_case(pkg, cuda, M, N, K, DTYPES[(M + N) % 3])


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_swiglu(pkg, cuda, M, N, K):
    print(f"case swiglu {M}x{N}x{K}", flush=True)
    _swiglu_case(pkg, cuda, M, N, K, DTYPES[(M + K) % 3])


@pytest.mark.parametrize("nmat,M,N,K", PLAN_SHAPES)
def test_every_planned_kernel(pkg, cuda, nmat, M, N, K):
    plan = (ctypes.c_int * 5)()
    assert pkg.lib().qmlp_w4a8_plan(M, N, K, nmat, 256, plan) == 0
    print(f"case plan {nmat} {M}x{N}x{K} {list(plan)}", flush=True)
    (_linear_case if nmat == 1 else _swiglu_case)(pkg, cuda, M, N, K, torch.bfloat16)


def test_rows_that_are_not_numbers_stay_apart(pkg, cuda):
    for M in (3, 40, 200):
        x = _rows(M, 512, torch.bfloat16, 5)
        w, _ = _weight(pkg, 96, 512, 6, cuda)
        clean = pkg.w4a8_linear(x.to(cuda), w)
        x[1, 77], x[M - 1, 500] = float("nan"), float("-inf")
        y = pkg.w4a8_linear(x.to(cuda), w)
        bad = torch.zeros(M, dtype=torch.bool)
        bad[[1, M - 1]] = True
        assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])


def test_widest_scales(pkg, cuda):
    """Blocks from the smallest step to the largest magnitude, saturation at 2^127 included."""
    x = torch.ones(6, 64)
    x[0] *= 2.0 ** -126
    x[1] *= 1e-45
    x[2] *= 3e38
    x[3, :32], x[3, 32:] = 2.0 ** 126, -(2.0 ** -100)
    x[4] = 0
    x[5] *= 2.0 ** 127
    t = pkg.quantize_mxint8(x.to(cuda))
    want = omi.quantize(x.double().numpy())
    for a, b in zip(_unpack(pkg, t), want):
        assert np.array_equal(a, b)
    assert np.array_equal(_np(pkg.dequantize(t)), omi.dequantize(*want))
    codes = np.full((32, 64), 1, dtype=np.uint8)  # .5
    scales = np.full((32, 2), 40, dtype=np.uint8)
    w = pkg.pack_canonical(torch.from_numpy(omx.join(codes)).to(cuda), torch.from_numpy(scales).to(cuda), "mxfp4")
    ref, mag = omx.linear(omi.dequantize(*want), omx.dequantize(codes, scales))
    y = _np(pkg.w4a8_linear(t, w, out_dtype=torch.float32))
    tiny = 2.0 ** -126  # below it a result may be flushed
    assert (np.abs(y - ref) <= _sum_error(64, mag) + tiny).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_products_of_strided_rows(pkg, cuda, dtype):
    """Rows apart in memory, quantised by the product and in front of it."""
    for M in (1, 2, 4, 16, 40):
        wide = _rows(M, 544, dtype, M).to(cuda)
        x = wide[:, :320]
        w, _ = _weight(pkg, 256, 320, 6, cuda)
        assert M == 1 or not x.is_contiguous()
        assert torch.equal(pkg.w4a8_linear(x, w), pkg.w4a8_linear(x.contiguous(), w))
        assert torch.equal(pkg.w4a8_swiglu(x, w, w), pkg.w4a8_swiglu(pkg.quantize_mxint8(x), w, w))


def test_offsets_beyond_32_bits(pkg, cuda):
    """A packed matrix of more than 2^32 bytes, its rows more than 2^32 bytes from the first: the last rows and columns,
    against the same rows by themselves."""
    rows, cols = 65536, 81920
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(rows, cols, generator=g, device=cuda, dtype=torch.bfloat16)
    t, last = pkg.quantize_mxint8(x), x[-96:]
    few = pkg.quantize_mxint8(last)
    assert t.nbytes > 1 << 32 and torch.equal(t.buf[-few.nbytes:], few.buf)
    n = torch.randn(cols, generator=g, device=cuda, dtype=torch.bfloat16)
    h, q = pkg.add_rmsnorm(x, x, n)
    h2, q2 = pkg.add_rmsnorm(last, last, n)
    assert torch.equal(h[-96:], h2) and torch.equal(q.buf[-few.nbytes:], q2.buf)
    del h, q
    codes = torch.randint(0, 256, (40, cols // 2), generator=g, device=cuda, dtype=torch.uint8)
    w = pkg.pack_canonical(codes, torch.full((40, cols // 32), 120, dtype=torch.uint8, device=cuda), "mxfp4")
    y = pkg.w4a8_linear(t, w, out_dtype=torch.float32)
    xd = pkg.dequantize(few).double()
    ref = (xd @ pkg.dequantize(w).double().T).cpu().numpy()
    mag = (xd.abs() @ pkg.dequantize(w).double().abs().T).cpu().numpy()
    assert (np.abs(_np(y[-96:]) - ref) <= _sum_error(cols, mag)).all()
    assert torch.equal(pkg.dequantize(t, dtype=torch.bfloat16)[-96:], pkg.dequantize(few, dtype=torch.bfloat16))


@pytest.mark.parametrize("rows,cols", [(1 << 20, 32), (2, 1 << 20)])
def test_largest_matrices(pkg, cuda, rows, cols):
    """Quantised, read back and behind the norm, against the oracle on some of their rows."""
    print(f"case largest {rows}x{cols}", flush=True)
    base = _rows(min(rows, 96), cols, torch.bfloat16, 9)
    x = base.to(cuda).repeat(-(-rows // 96), 1)[:rows].contiguous()
    t = pkg.quantize_mxint8(x)
    q, scales = pkg.unpack_canonical(t)
    want, wants = omi.quantize(_np(base))
    assert np.array_equal(q[:96].cpu().numpy(), want) and np.array_equal(scales[:96].cpu().numpy(), wants)
    for at in (range(96, rows - 95, 96 * 1021) if rows > 96 else ()):
        assert torch.equal(q[at:at + 96], q[:96]) and torch.equal(scales[at:at + 96], scales[:96])
    assert torch.equal(q[-1], q[(rows - 1) % 96]) and torch.equal(scales[-1], scales[(rows - 1) % 96])
    values = pkg.dequantize(t)
    assert torch.equal(values, (q.float().view(rows, -1, 32) * torch.exp2(scales.float() - 133)[..., None]).view(rows, cols))
    w = torch.zeros(cols, dtype=torch.bfloat16, device=cuda)
    h, n, normed = pkg.add_rmsnorm(x, x, w, output="both")
    few = pkg.add_rmsnorm(x[:96], x[:96], w, output="both")
    assert torch.equal(h, 2 * x)
    for a, b in ((n, few[1]), *zip(pkg.unpack_canonical(normed), pkg.unpack_canonical(few[2]))):
        assert torch.equal(a[:96], b) and torch.equal(a[-1], b[(rows - 1) % 96])


@pytest.mark.parametrize("M,N,K", [(1, 1 << 20, 64), (9, 1 << 20, 64), (70, 1 << 20, 64), (1, 33, 1 << 20), (12, 33, 1 << 20),
                                   (40, 33, 1 << 20), (300, 33, 1 << 20)])
def test_products_at_the_largest_sizes(pkg, cuda, M, N, K):
    """Every block's step is the same and so is every weight's scale, so every product is a whole number of half steps
    of at most 127 * 12 units.  A random sum of 2^20 of them (a spread of 2^10 times 450 or so) stays below 2^22 units, a
    digit's part of it too, so no sum rounds.  Behind it the silu's error as elsewhere."""
    print(f"case largest product {M}x{N}x{K}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(N)
    q = torch.randint(-127, 128, (M, K), generator=g, device=cuda).float()
    q[:, ::32] = 127.0
    x = q / 64
    t = pkg.quantize_mxint8(x)
    assert torch.equal(pkg.dequantize(t), x)
    byte = 127 - (K.bit_length() - 1) // 2  # the sums have a spread of a few units

    def weight():
        codes = torch.randint(0, 256, (N, K // 2), generator=g, device=cuda, dtype=torch.uint8)
        return pkg.pack_canonical(codes, torch.full((N, K // 32), byte, dtype=torch.uint8, device=cuda), "mxfp4")

    w1, w3 = weight(), weight()
    y1, y3 = (x.double() @ pkg.dequantize(w).double().T.contiguous() for w in (w1, w3))
    for a in (x, t):
        for w, y in ((w1, y1), (w3, y3)):
            assert torch.equal(pkg.w4a8_linear(a, w, out_dtype=torch.float32).double(), y)
    s = y1 / (1 + torch.exp(-y1)) * y3
    got = pkg.w4a8_swiglu(t, w1, w3, out_dtype=torch.float32).double()
    assert ((got - s).abs() <= (8 + y1.abs()) * 2.0 ** -23 * s.abs() + 1.1e-36 * y3.abs()).all()
