"""Microscaled 4-bit floating point (OCP MXFP4): the activations' side of the format and the products.

32 consecutive K values share one power-of-two scale byte, each value is one of 0, .5, 1, 1.5, 2, 3, 4,
6 with a sign.  A block's scale is the binade of its largest magnitude less 2 (at least 2^-126); values
are rounded half to even and saturate at 6; a block that holds an infinity or a NaN becomes NaN.

* ``quantize_mxfp4(x)`` -> ``MxTensor``, a packed activation matrix that feeds any number of products
  (``dequantize`` and ``unpack_canonical`` take it too);
* ``mxfp4_linear(x, w, residual=...)``: ``out = x w^T (+ residual)``;
* ``mxfp4_swiglu(x, w1, w3)``: ``silu(x w1^T) * (x w3^T)``, the gate/up pair of the block, as rows or
  (``quantize=True``) as the ``MxTensor`` that the down projection takes.

``x`` is an ``MxTensor`` or a bf16, fp16 or fp32 ``[M, K]`` tensor, which the call quantises; weights come
from ``pack_weight(w, "mxfp4")`` or, for checkpoints that hold the format, ``pack_canonical(codes, scales,
"mxfp4")``.  Sizes: any M up to 65536 and any N, K a multiple of 32.  The reference's counterparts are the
4-bit linears of its block (``docker/qwen-c2-graft/graft/mlp.py:17-19,402-423``) and the fused gate/up
projection (``scripts/ci/fused_1d.py:123-196``).

Every call runs on the inputs' GPU, on ``stream`` or that GPU's current stream, may be captured into a
HIP graph and allocates its output and scratch memory from torch's caching allocator there.  Errors:
``ValueError`` for wrong shapes, dtypes or devices, ``QmlpError`` for launch failures.
"""
import functools
from dataclasses import dataclass

import torch

from . import _lib
from .mlp import PackedWeight, _check_device_tensor, _check_mxfp4_buffer, _mxfp4_bytes, _same_device

_X_TYPES = {torch.bfloat16: _lib.X_BF16, torch.float16: _lib.X_F16, torch.float32: _lib.X_F32}


@dataclass
class MxTensor:
    """A packed MXFP4 activation matrix ``[rows, cols]`` (device bytes + shape)."""

    buf: torch.Tensor  # uint8, qmlp_packed_bytes(rows, cols, QMLP_FMT_MXFP4) bytes
    rows: int
    cols: int

    fmt = "mxfp4"
    fmt_code = _lib.FMT_MXFP4

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self):
        return self.buf.device

    @property
    def nbytes(self):
        return self.buf.numel()

    def data_ptr(self):
        return self.buf.data_ptr()


def _check_rows(x):
    """(QMLP_X_* code, row stride) of a 2-D GPU tensor whose rows are contiguous; the rows themselves may
    be strided."""
    if not isinstance(x, torch.Tensor):
        raise ValueError("x must be a torch.Tensor or an MxTensor")
    if not x.is_cuda:
        raise ValueError(f"x must be on the GPU, got {x.device}")
    x_type = _X_TYPES.get(x.dtype)
    if x_type is None:
        raise ValueError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() != 2 or 0 in x.shape:
        raise ValueError(f"x must be a non-empty 2-D tensor, got {tuple(x.shape)}")
    rows, cols = x.shape
    if cols % 32:
        raise ValueError(f"x must have a multiple of 32 columns (the format's block), got {cols}")
    stride, step = x.stride()
    if step != 1:
        raise ValueError("x must have contiguous rows")
    if rows == 1:
        stride = cols
    if stride < cols or stride * (4 if x_type == _lib.X_F32 else 2) % 16 or x.data_ptr() % 16:
        raise ValueError(f"x: rows must start at multiples of 16 bytes and not overlap (stride {stride})")
    return x_type, stride


def quantize_mxfp4(x, norm_weight=None, eps=1e-6, stream=None):
    """bf16, fp16 or fp32 ``[M, K]`` GPU tensor (rows may be strided) -> ``MxTensor``.

    With ``norm_weight`` (bf16 ``[K]``, x bf16) the decoder's zero-centred RMSNorm runs in front, in the
    same pass: ``n = bf16(rmsnorm(x) * (1 + norm_weight))`` is what is quantised.
    """
    x_type, stride = _check_rows(x)
    M, K = x.shape
    if norm_weight is not None:
        _check_device_tensor(norm_weight, "norm_weight", torch.bfloat16)
        if x.dtype != torch.bfloat16:
            raise ValueError("x must be bf16 in front of a norm")
        if tuple(norm_weight.shape) != (K,):
            raise ValueError(f"norm_weight must have shape ({K},)")
        _same_device(x.device, norm_weight=norm_weight)
    device, nbytes = x.device, _mxfp4_bytes(M, K)
    with _lib.on_device(device, stream):
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        if norm_weight is None:
            rc = _lib.lib().qmlp_mx_quantize(x.data_ptr(), x_type, stride, M, K, buf.data_ptr(), nbytes,
                                             _lib.device_stream(device, stream))
        else:
            rc = _lib.lib().qmlp_mx_quantize_rmsnorm(x.data_ptr(), stride, norm_weight.data_ptr(), float(eps), M, K,
                                                     buf.data_ptr(), nbytes, _lib.device_stream(device, stream))
        _lib.check(rc, "quantize_mxfp4")
    return MxTensor(buf, M, K)


def _check_buffers(x, **weights):
    if isinstance(x, MxTensor):
        _check_mxfp4_buffer(x, "x")
    for name, w in weights.items():
        _check_mxfp4_buffer(w, name)


def _check_weight(w, name, K):
    if not isinstance(w, PackedWeight) or w.fmt != "mxfp4":
        raise ValueError(f'{name} must be a PackedWeight in the "mxfp4" format')
    if w.cols != K:
        raise ValueError(f"{name} has {w.cols} columns, x has {K}")


def _activation(x):
    """(pointer, QMLP_X_* code, row stride, M, K, device) of an activation argument."""
    if isinstance(x, MxTensor):
        return x.buf.data_ptr(), _lib.X_MXFP4, 0, x.rows, x.cols, x.buf.device
    x_type, stride = _check_rows(x)
    M, K = x.shape
    return x.data_ptr(), x_type, stride, M, K, x.device


def _check_out(out, out_dtype, shape):
    if out is None:
        if out_dtype not in (None, torch.bfloat16, torch.float32):
            raise ValueError("out_dtype must be bf16 or fp32")
        return torch.bfloat16 if out_dtype is None else out_dtype
    _check_device_tensor(out, "out")
    if out.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("out must be bf16 or fp32")
    if out_dtype not in (None, out.dtype):
        raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
    if tuple(out.shape) != shape:
        raise ValueError(f"out must have shape {shape}")
    return out.dtype


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(M, N, K, x_type):
    return _lib.lib().qmlp_mx_workspace_bytes(M, N, K, x_type)


def _workspace(M, N, K, x_type, device):
    """(tensor that has to live until the call is enqueued, pointer, bytes); none where none is needed."""
    n = _workspace_bytes(M, N, K, x_type)
    if n == 0:
        return None, None, 0
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def mxfp4_linear(x, w, residual=None, out=None, out_dtype=None, stream=None):
    """``out = x w^T (+ residual)`` with both operands in MXFP4 and fp32 sums.

    ``x``: ``MxTensor`` or bf16 / fp16 / fp32 ``[M, K]`` (quantised in the call); ``w``: mxfp4
    ``PackedWeight`` ``[N, K]``; ``residual`` bf16 or fp32 ``[M, N]``; ``out`` (or ``out_dtype`` when
    ``out`` is None) bf16, rounded once to nearest-even, or fp32.  ``out`` may be the residual itself.
    """
    xp, x_type, stride, M, K, device = _activation(x)
    _check_weight(w, "w", K)
    shape = (M, w.rows)
    dtype = _check_out(out, out_dtype, shape)
    flags = _lib.OUT_F32 if dtype == torch.float32 else 0
    if residual is not None:
        _check_device_tensor(residual, "residual")
        if residual.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("residual must be bf16 or fp32")
        if tuple(residual.shape) != shape:
            raise ValueError(f"residual must have shape {shape}")
        if residual.dtype == torch.float32:
            flags |= _lib.RESIDUAL_F32
    _check_buffers(x, w=w)
    _same_device(device, w=w.buf, residual=residual, out=out)
    with _lib.on_device(device, stream):
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=device)
        ws, wp, wn = _workspace(M, w.rows, K, x_type, device)
        rc = _lib.lib().qmlp_mx_linear(xp, x_type, stride, w.buf.data_ptr(),
                                       None if residual is None else residual.data_ptr(), out.data_ptr(), wp, wn, M,
                                       w.rows, K, flags, _lib.device_stream(device, stream))
        _lib.check(rc, "mxfp4_linear")
    return out


def mxfp4_swiglu(x, w1, w3, out=None, out_dtype=None, quantize=False, stream=None):
    """``silu(x w1^T) * (x w3^T)`` with every operand in MXFP4 and fp32 sums.

    ``x`` as in ``mxfp4_linear``; ``w1`` (gate) and ``w3`` (up): mxfp4 ``PackedWeight`` ``[N, K]``.  The
    result is a bf16 or fp32 ``[M, N]`` tensor (``out`` / ``out_dtype``) or, with ``quantize=True`` (N a
    multiple of 256), an ``MxTensor``, quantised from the fp32 values.
    """
    xp, x_type, stride, M, K, device = _activation(x)
    _check_weight(w1, "w1", K)
    _check_weight(w3, "w3", K)
    N = w1.rows
    if w3.rows != N:
        raise ValueError(f"w1 has {N} rows, w3 {w3.rows}")
    if quantize:
        if out is not None or out_dtype is not None:
            raise ValueError("quantize=True makes its own MxTensor: out and out_dtype do not apply")
        if N % 256:
            raise ValueError(f"quantize=True needs N to be a multiple of 256, got {N}")
        flags = _lib.OUT_MXFP4
    else:
        dtype = _check_out(out, out_dtype, (M, N))
        flags = _lib.OUT_F32 if dtype == torch.float32 else 0
    _check_buffers(x, w1=w1, w3=w3)
    _same_device(device, w1=w1.buf, w3=w3.buf, out=out)
    with _lib.on_device(device, stream):
        if quantize:
            res = MxTensor(torch.empty(_mxfp4_bytes(M, N), dtype=torch.uint8, device=device), M, N)
            out = res.buf
        else:
            out = res = torch.empty((M, N), dtype=dtype, device=device) if out is None else out
        ws, wp, wn = _workspace(M, N, K, x_type, device)
        rc = _lib.lib().qmlp_mx_swiglu(xp, x_type, stride, w1.buf.data_ptr(), w3.buf.data_ptr(), out.data_ptr(), wp, wn,
                                       M, N, K, flags, _lib.device_stream(device, stream))
        _lib.check(rc, "mxfp4_swiglu")
    return res
