"""The tiled MXFP4 kernels on the GPU: every height, whole and in K pieces, with a last tile of features that
is full and one that is not; what they write beside their outputs, rows that are not numbers, extreme
scales, replayed graphs, streams at once, and the block on them.  Each test asserts that its sizes are
planned on tiles."""
import os
import subprocess
import sys

import numpy as np
import pytest
import test_gpu_mxfp4 as mx
import torch
from test_mxfp4 import TILE_SHAPES, tile_plan

from oracle import mxfp4 as omx

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FILL = 0x5A
MARGIN = 1 << 16  # guard bytes on either side of a buffer

# (matrices, M, N, K, in pieces)
FEW = [(1, 1107, 65, 96, False), (1, 1097, 66, 3904, True), (1, 1361, 8237, 96, False), (2, 33, 250, 22816, True),
       (2, 1178, 3331, 96, False), (2, 65, 2803, 16352, True)]


def _planned(pkg, nmat, M, N, K, split):
    height, ks = tile_plan(pkg, nmat, M, N, K)
    assert (ks > 1) == split, (nmat, M, N, K, height, ks)


def _operands(pkg, cuda, nmat, M, N, K, dtype=torch.bfloat16):
    x = mx._rows(M, K, dtype, M + K).to(cuda)
    g = torch.Generator(device=cuda).manual_seed(N)
    w = [pkg.pack_canonical(torch.randint(0, 256, (N, K // 2), generator=g, device=cuda, dtype=torch.uint8),
                            torch.randint(116, 122, (N, K // 32), generator=g, device=cuda, dtype=torch.uint8), "mxfp4")
         for _ in range(nmat)]
    return x, w


def _product(pkg, x, w, **kw):
    return pkg.mxfp4_linear(x, *w, **kw) if len(w) == 1 else pkg.mxfp4_swiglu(x, *w, **kw)


@pytest.mark.parametrize("nmat,M,N,K", TILE_SHAPES)
def test_every_tiled_kernel(pkg, cuda, nmat, M, N, K):
    tile_plan(pkg, nmat, M, N, K)
    mx.test_every_planned_kernel(pkg, cuda, nmat, M, N, K)


# ---------------------------------------------------------------- what is written


class _Guarded:
    """``n`` device bytes between two margins, all of them FILL."""

    def __init__(self, n, cuda):
        self.flat = torch.full((n + 2 * MARGIN,), FILL, dtype=torch.uint8, device=cuda)
        self.view = self.flat[MARGIN:MARGIN + n]

    def intact(self):
        return bool((self.flat[:MARGIN] == FILL).all()) and bool((self.flat[MARGIN + self.view.numel():] == FILL).all())


def _written(M, K):
    """Which bytes of a packed activation matrix of M rows hold them (K up to a unit's end included)."""
    tiles, units = -(-M // 32), -(-K // 256)
    b = np.zeros((tiles, units, 4352), dtype=bool)
    for r in range(M):
        u, r = b[r // 32], r % 32
        for kb in range(8):
            u[:, (kb * 32 + r) * 16:(kb * 32 + r) * 16 + 16] = True
        for h in (0, 32):
            u[:, 4096 + 4 * (r + h):4096 + 4 * (r + h) + 4] = True
    return b.reshape(-1)


@pytest.mark.parametrize("nmat,M,N,K,split", FEW + [(2, 33, 256, 22816, True), (2, 1178, 3328, 96, False)])
def test_products_write_their_output_and_workspace_only(pkg, cuda, nmat, M, N, K, split):
    from qwen_mlp_amd import _lib

    print(f"case guards nmat={nmat} {M}x{N}x{K}", flush=True)
    _planned(pkg, nmat, M, N, K, split)
    lib = pkg.lib()
    x, w = _operands(pkg, cuda, nmat, M, N, K)
    need = lib.qmlp_mx_workspace_bytes(M, N, K, _lib.X_BF16)
    outs = [("fp32", 4 * M * N, _lib.OUT_F32, torch.float32), ("bf16", 2 * M * N, 0, torch.bfloat16)]
    if nmat == 2 and N % 256 == 0:
        outs.append(("packed", omx.packed_bytes(M, N) - omx.TRAILER_BYTES, _lib.OUT_MXFP4, None))
    for name, nbytes, flags, dtype in outs:
        ws, out = _Guarded(need, cuda), _Guarded(nbytes, cuda)
        args = [_lib.ptr(x), _lib.X_BF16, K, *(_lib.ptr(v.buf) for v in w)]
        args += [None] if nmat == 1 else []
        fn = lib.qmlp_mx_linear if nmat == 1 else lib.qmlp_mx_swiglu
        _lib.check(fn(*args, _lib.ptr(out.view), _lib.ptr(ws.view), need, M, N, K, flags, _lib.stream_handle()), name)
        torch.cuda.synchronize()
        assert ws.intact() and out.intact(), name
        if dtype is None:
            got = out.view.cpu().numpy()
            want = pkg.mxfp4_swiglu(x, *w, quantize=True).buf.cpu().numpy()
            mask = _written(M, N)
            assert np.array_equal(got[mask], want[:got.size][mask]) and (got[~mask] == FILL).all()
        else:
            assert torch.equal(out.view.view(dtype).view(M, N), _product(pkg, x, w, out_dtype=dtype))


@pytest.mark.parametrize("rows,cols", [(1, 32), (33, 288), (1030, 8320), (40, 17408)])
def test_quantisation_writes_its_rows_only(pkg, cuda, rows, cols):
    from qwen_mlp_amd import _lib

    lib, mask = pkg.lib(), _written(rows, cols)
    x = mx._rows(rows, cols, torch.bfloat16, rows).to(cuda)
    norm = torch.zeros(cols, dtype=torch.bfloat16, device=cuda)
    n = omx.packed_bytes(rows, cols) - omx.TRAILER_BYTES
    for normed in (False, True):
        out = _Guarded(n, cuda)
        if normed:
            rc = lib.qmlp_mx_quantize_rmsnorm(_lib.ptr(x), cols, _lib.ptr(norm), 1e-6, rows, cols, _lib.ptr(out.view), n,
                                              _lib.stream_handle())
        else:
            rc = lib.qmlp_mx_quantize(_lib.ptr(x), _lib.X_BF16, cols, rows, cols, _lib.ptr(out.view), n,
                                      _lib.stream_handle())
        _lib.check(rc, "quantise")
        got = out.view.cpu().numpy()
        want = pkg.quantize_mxfp4(x, norm_weight=norm if normed else None).buf.cpu().numpy()
        assert out.intact() and (got[~mask] == FILL).all() and np.array_equal(got[mask], want[:n][mask])


def test_the_block_writes_its_output_and_workspace_only(pkg, cuda):
    """Also the arrival counters of the other formats, in front, stay zero."""
    from qwen_mlp_amd import _lib

    H, I, M = 256, 4096, 1100
    _planned(pkg, 2, M, I, H, False)
    _planned(pkg, 1, M, H, I, True)
    w = pkg.load_mlp_weights(cuda, mx._state_dict(H, I, cuda), weight_format="mxfp4")
    x = mx._rows(M, H, torch.bfloat16, 3, 0.05).to(cuda)
    need = pkg.workspace_bytes(M, H, I, "mxfp4")
    ws, out = _Guarded(need, cuda), _Guarded(2 * M * H, cuda)
    _lib.check(pkg.lib().qmlp_workspace_init(_lib.ptr(ws.view), need, _lib.stream_handle()), "init")
    y = pkg.mlp_forward(x, w, residual=x, out=out.view.view(torch.bfloat16).view(M, H), workspace=ws.view)
    assert torch.equal(y, pkg.mlp_forward(x, w, residual=x))
    assert ws.intact() and out.intact() and not ws.view[:_lib.WS_COUNTER_BYTES].any()


# ---------------------------------------------------------------- values


@pytest.mark.parametrize("nmat,M,N,K,split", FEW)
def test_rows_that_are_not_numbers_stay_in_their_row(pkg, cuda, nmat, M, N, K, split):
    print(f"case nan nmat={nmat} {M}x{N}x{K}", flush=True)
    _planned(pkg, nmat, M, N, K, split)
    x, w = _operands(pkg, cuda, nmat, M, N, K, torch.float32)
    clean = _product(pkg, x, w, out_dtype=torch.float32)
    bad = [1, M // 2, M - 1]
    for row, value in zip(bad, (float("inf"), -float("inf"), float("nan"))):
        x[row, (37 * row) % K] = value
    y = _product(pkg, x, w, out_dtype=torch.float32)
    rest = torch.ones(M, dtype=torch.bool, device=cuda)
    rest[bad] = False
    assert torch.isnan(y[bad]).all() and torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("byte", [0, 1, 64, 127, 200, 225])
@pytest.mark.parametrize("M,N,K,split", [(1107, 65, 96, False), (1097, 66, 3904, True)])
def test_scales_over_their_whole_range(pkg, cuda, byte, M, N, K, split):
    """|x| <= 2^8 and a weight is at most 6 2^(byte - 127), so that no sum of 3904 products reaches
    2^(12 + 8 + 3 + byte - 127) < 2^127.  On top of the sums' rounding each product, and each of at most as
    many sums, may lose what is below the smallest normal number, 2^-126."""
    _planned(pkg, 1, M, N, K, split)
    codes = np.random.default_rng(byte).integers(0, 16, (N, K), dtype=np.uint8)
    scales = np.full((N, K // 32), byte, dtype=np.uint8)
    w = pkg.pack_canonical(torch.from_numpy(omx.join(codes)).to(cuda), torch.from_numpy(scales).to(cuda), "mxfp4")
    x = mx._rows(M, K, torch.float32, M).clamp(-256, 256)
    ref, mag = omx.linear(omx.dequantize(*omx.quantize(x.double().numpy())), omx.dequantize(codes, scales))
    y = pkg.mxfp4_linear(x.to(cuda), w, out_dtype=torch.float32)
    assert (np.abs(mx._np(y) - ref) <= mx._sum_error(K, mag) + 2 * K * 2.0 ** -126).all()


# ---------------------------------------------------------------- graphs, streams


@pytest.mark.parametrize("nmat,M,N,K,split", [(1, 1107, 65, 96, False), (1, 1097, 66, 3904, True),
                                              (2, 33, 256, 22816, True), (2, 1178, 3328, 96, False)])
def test_graph_replays(pkg, cuda, nmat, M, N, K, split):
    _planned(pkg, nmat, M, N, K, split)
    x, w = _operands(pkg, cuda, nmat, M, N, K)
    down = _operands(pkg, cuda, 1, 1, 96, N)[1] if nmat == 2 else None

    def chain(v):
        if nmat == 1:
            return pkg.mxfp4_linear(v, *w, out_dtype=torch.float32)
        return pkg.mxfp4_linear(pkg.mxfp4_swiglu(v, *w, quantize=True), *down, out_dtype=torch.float32)

    static = x.clone()
    for _ in range(2):
        chain(static)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = chain(static)
        graphs.append((g, y))
    for i in range(4):
        new = mx._rows(M, K, torch.bfloat16, 50 + i).to(cuda)
        eager = chain(new)
        static.copy_(new)
        for g, y in graphs:
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
            torch.empty(1 << 20, device=cuda).fill_(1.0)


def test_a_first_call_may_be_captured():
    """In a fresh process, products whose kernels have not run before, captured without a warm-up call."""
    code = f"""
import sys
sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, "tests")!r}]
import torch
import __graft_entry__
pkg = __graft_entry__.load_package()
import test_gpu_mxfp4_tiles as t
dev = torch.device("cuda:0")
cases = [t._operands(pkg, dev, *c[:4]) for c in t.FEW]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = [t._product(pkg, x, w) for x, w in cases]
g.replay()
torch.cuda.synchronize()
print("RESULT", [bool(torch.equal(y, t._product(pkg, x, w))) for y, (x, w) in zip(got, cases)], flush=True)
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=110)
    assert res.returncode == 0 and f"RESULT {[True] * len(FEW)}" in res.stdout, res.stdout + res.stderr


def test_two_streams_at_once(pkg, cuda):
    """Split products on two streams, each with partial tiles of its own."""
    sizes = [(1, 1097, 66, 3904), (2, 65, 2816, 16352)]
    for c in sizes:
        _planned(pkg, *c, True)
    cases = [_operands(pkg, cuda, *c) for c in sizes]
    want = [_product(pkg, x, w, out_dtype=torch.float32) for x, w in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(10):
        for k, (s, (x, w)) in enumerate(zip(streams, cases)):
            if i % 2:
                with torch.cuda.stream(s):
                    got[k].append(_product(pkg, x, w, out_dtype=torch.float32))
            else:
                got[k].append(_product(pkg, x, w, out_dtype=torch.float32, stream=s))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(y, want[k]) for y in got[k])


# ---------------------------------------------------------------- the block

# (H, I, M, gate/up in pieces, down in pieces)
BLOCKS = [(256, 512, 1100, False, False), (512, 2048, 1100, False, False), (256, 4096, 1100, False, True),
          (256, 16384, 1500, False, True), (16384, 512, 130, True, False), (8192, 6144, 65, True, True)]


@pytest.mark.parametrize("H,I,M,gate_up,down", BLOCKS)
def test_block(pkg, cuda, H, I, M, gate_up, down):
    _planned(pkg, 2, M, I, H, gate_up)
    _planned(pkg, 1, M, H, I, down)
    mx.test_block(pkg, cuda, H, I, M)


def test_pool_shared_with_other_formats(pkg, cuda):
    """Forwards on tiles in a workspace that the formats that count arrivals in it use in turn."""
    H, I, M, many = 512, 8192, 16, 1100
    _planned(pkg, 2, many, I, H, False)
    _planned(pkg, 1, many, H, I, True)
    sd = mx._state_dict(H, I, cuda)
    pool = pkg.WorkspacePool()
    mlps = [pkg.Qwen36MLP(cuda, sd, weight_format=f, max_tokens=many, pool=pool) for f in ("bfp8", "mxfp4", "bf16")]
    x = mx._rows(M, H, torch.bfloat16, 3, 0.05).to(cuda)
    big = mx._rows(many, H, torch.bfloat16, 4, 0.05).to(cuda)
    first = [(m.forward(x), m.forward(big)) for m in mlps]
    for _ in range(3):
        for m, (few, all_) in zip(mlps, first):
            assert torch.equal(m.forward(big), all_)
            assert torch.equal(m.forward(x), few)
