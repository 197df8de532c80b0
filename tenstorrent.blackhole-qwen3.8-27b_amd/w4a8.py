"""4-bit weights with 8-bit activations: MXFP4 matrices multiplied by activations in MXINT8, and the norm with
the residual's addition in front of them.

MXINT8 (OCP MX): 32 consecutive K values share a power-of-two scale and each is an integer of at most 127
steps; the step is a 64th of the binade of the block's largest magnitude (between 2^-126 and 2^120), values
are rounded half to even, 128 steps to 127.  A block that holds an infinity or a NaN becomes NaN.

* ``quantize_mxint8(x)`` -> ``Mx8Tensor``, a packed activation matrix that feeds any number of products
  (``dequantize`` and ``unpack_canonical`` take it too);
* ``add_rmsnorm(x, residual, norm_weight)`` -> ``(h, n)``: the residual's addition and the decoder's norm of
  the sum in one pass, ``n`` as an ``Mx8Tensor``, as bf16 rows, or both;
* ``w4a8_linear(x, w, residual=...)``: ``out = x w^T (+ residual)``;
* ``w4a8_swiglu(x, w1, w3)``: ``silu(x w1^T + gate_add) * (x w3^T + up_add)``, the gate/up pair of the block, as
  rows or (``quantize=True``) as the ``Mx8Tensor`` that the down projection takes;
* ``w4a8_mlp(x, weights, ...)``: the block of the two, with the adapters of many requests beside its projections
  (``Qwen36MLP(..., weight_format="mxfp4", activation_format="mxint8")`` calls it).

``x`` of the products is an ``Mx8Tensor`` or a bf16, fp16 or fp32 ``[M, K]`` tensor, which the call quantises;
weights come from ``pack_weight(w, "mxfp4")`` or ``pack_canonical(codes, scales, "mxfp4")``.  Sizes: any M up
to 65536 and any N, K a multiple of 32.  The reference's counterparts are the linears of its block
(``docker/qwen-c2-graft/graft/mlp.py:17-19,402-423``), the fused gate/up projection
(``scripts/ci/fused_1d.py:123-196``) and the decoder's add and norm (``layer.py:352-357``).

Every call runs on the inputs' GPU, on ``stream`` or that GPU's current stream, may be captured into a HIP
graph and allocates its output and scratch memory from torch's caching allocator there.  Errors: ``ValueError``
for wrong shapes, dtypes or devices, ``QmlpError`` for launch failures.
"""
import functools
from dataclasses import dataclass

import torch

from . import _lib
from .lora import lora_linear
from .mlp import _check_device_tensor, _check_mxfp4_buffer, _check_mxint8_buffer, _mxint8_bytes, _same_device
from .mxfp4 import _check_out, _check_rows, _check_weight


@dataclass
class Mx8Tensor:
    """A packed MXINT8 activation matrix ``[rows, cols]`` (device bytes + shape)."""

    buf: torch.Tensor  # uint8, qmlp_mxint8_bytes(rows, cols) bytes
    rows: int
    cols: int

    fmt = "mxint8"

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


def quantize_mxint8(x, stream=None):
    """bf16, fp16 or fp32 ``[M, K]`` GPU tensor (rows may be strided) -> ``Mx8Tensor``."""
    x_type, stride = _check_rows(x)
    M, K = x.shape
    device, nbytes = x.device, _mxint8_bytes(M, K)
    with _lib.on_device(device, stream):
        buf = x.new_empty(nbytes, dtype=torch.uint8)
        rc = _lib.lib().qmlp_mxint8_quantize(x.data_ptr(), x_type, stride, M, K, buf.data_ptr(), nbytes,
                                             _lib.device_stream(device, stream))
        _lib.check(rc, "quantize_mxint8")
    return Mx8Tensor(buf, M, K)


def _check_norm_rows(t, name):
    """(QMLP_X_* code, row stride) of a bf16 or fp32 ``[M, K]`` tensor with contiguous rows."""
    try:
        rows = _check_rows(t)
    except ValueError as e:
        raise ValueError(f"{name}: {e}") from None
    if rows[0] == _lib.X_F16:
        raise ValueError(f"{name} must be bf16 or fp32, got {t.dtype}")
    return rows


def add_rmsnorm(x, residual, norm_weight, eps=1e-6, output="mxint8", out=None, stream=None):
    """``h = residual + x``, ``n = bf16(rmsnorm(h) * (1 + norm_weight))`` -> ``(h, n)``.

    ``x`` (what attention or a feed-forward block returns) and ``residual`` (the residual stream) are bf16 or
    fp32 ``[M, K]``, rows may be strided; ``norm_weight`` bf16 ``[K]``.  ``h`` has the residual's dtype, to which
    the sum is rounded before the norm; it is written to ``out``, which may be the residual itself, or to a new
    tensor.  ``residual=None``: nothing is added, and ``h`` is ``x``.

    ``output``: "mxint8" -- ``n`` is an ``Mx8Tensor``, the quantisation of the bf16 rows; "rows" -- ``n`` is a
    bf16 tensor; "both" -- ``(h, n_rows, n_quantised)``, for a block whose adapters read the rows.
    """
    if output not in ("mxint8", "rows", "both"):
        raise ValueError(f'output must be "mxint8", "rows" or "both", got {output!r}')
    x_type, x_stride = _check_norm_rows(x, "x")
    M, K = x.shape
    device = x.device
    _check_device_tensor(norm_weight, "norm_weight", torch.bfloat16)
    if norm_weight.dim() != 1 or norm_weight.shape[0] != K:
        raise ValueError(f"norm_weight must have shape ({K},)")
    rp = hp = n = buf = np = bp = None
    r_type, r_stride, h_stride, nbytes = x_type, 0, 0, 0
    if residual is not None:
        r_type, r_stride = _check_norm_rows(residual, "residual")
        if residual.shape != x.shape:
            raise ValueError(f"residual must have shape ({M}, {K})")
        rp = residual.data_ptr()
        if out is not None:
            h_type, h_stride = _check_norm_rows(out, "out")
            if h_type != r_type or out.shape != x.shape:
                raise ValueError(f"out must be a {residual.dtype} tensor of shape ({M}, {K})")
    elif out is not None:
        raise ValueError("out is the sum with a residual: none is written without one")
    _same_device(device, norm_weight=norm_weight, residual=residual, out=out)
    with _lib.on_device(device, stream):
        h = x
        if residual is not None:
            h = out
            if h is None:
                h, h_stride = residual.new_empty((M, K)), K
            hp = h.data_ptr()
        if output != "mxint8":
            n = x.new_empty((M, K), dtype=torch.bfloat16)
            np = n.data_ptr()
        if output != "rows":
            nbytes = _mxint8_bytes(M, K)
            buf = x.new_empty(nbytes, dtype=torch.uint8)
            bp = buf.data_ptr()
        rc = _lib.lib().qmlp_add_rmsnorm(x.data_ptr(), x_type, x_stride, rp, r_type, r_stride, norm_weight.data_ptr(),
                                         float(eps), M, K, hp, h_stride, np, bp, nbytes,
                                         _lib.device_stream(device, stream))
        _lib.check(rc, "add_rmsnorm")
    if output == "rows":
        return h, n
    q = Mx8Tensor(buf, M, K)
    return (h, q) if output == "mxint8" else (h, n, q)


def _activation(x):
    """(pointer, QMLP_X_* code, row stride, M, K, device) of an activation argument."""
    if isinstance(x, Mx8Tensor):
        _check_mxint8_buffer(x, "x")
        return x.buf.data_ptr(), _lib.X_MXINT8, 0, x.rows, x.cols, x.buf.device
    x_type, stride = _check_rows(x)
    M, K = x.shape
    return x.data_ptr(), x_type, stride, M, K, x.device


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(M, N, K, x_type):
    return _lib.lib().qmlp_w4a8_workspace_bytes(M, N, K, x_type)


def _workspace(M, N, K, x_type, device):
    """(tensor that has to live until the call is enqueued, pointer, bytes); none where none is needed."""
    n = _workspace_bytes(M, N, K, x_type)
    if n == 0:
        return None, None, 0
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def w4a8_linear(x, w, residual=None, out=None, out_dtype=None, stream=None):
    """``out = x w^T (+ residual)`` with x in MXINT8, w in MXFP4 and fp32 sums.

    ``x``: ``Mx8Tensor`` or bf16 / fp16 / fp32 ``[M, K]`` (quantised in the call); ``w``: mxfp4
    ``PackedWeight`` ``[N, K]``; ``residual`` bf16 or fp32 ``[M, N]`` (what ``lora_linear`` returns, beside
    the residual stream); ``out`` (or ``out_dtype`` when ``out`` is None) bf16, rounded once to nearest-even, or
    fp32.  ``out`` may be the residual itself.
    """
    xp, x_type, stride, M, K, device = _activation(x)
    _check_weight(w, "w", K)
    _check_mxfp4_buffer(w, "w")
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
    _same_device(device, w=w.buf, residual=residual, out=out)
    with _lib.on_device(device, stream):
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=device)
        ws, wp, wn = _workspace(M, w.rows, K, x_type, device)
        rc = _lib.lib().qmlp_w4a8_linear(xp, x_type, stride, w.buf.data_ptr(),
                                         None if residual is None else residual.data_ptr(), out.data_ptr(), wp, wn, M,
                                         w.rows, K, flags, _lib.device_stream(device, stream))
        _lib.check(rc, "w4a8_linear")
    return out


def w4a8_swiglu(x, w1, w3, gate_add=None, up_add=None, out=None, out_dtype=None, quantize=False, stream=None):
    """``silu(x w1^T + gate_add) * (x w3^T + up_add)`` with x in MXINT8, the weights in MXFP4 and fp32 sums.

    ``x`` as in ``w4a8_linear``; ``w1`` (gate) and ``w3`` (up): mxfp4 ``PackedWeight`` ``[N, K]``; ``gate_add``,
    ``up_add``: fp32 ``[M, N]`` (what ``lora_linear`` returns for the two projections) or None.  The result is a
    bf16 or fp32 ``[M, N]`` tensor (``out`` / ``out_dtype``) or, with ``quantize=True`` (N a multiple of 256), an
    ``Mx8Tensor``, quantised from the fp32 values.
    """
    xp, x_type, stride, M, K, device = _activation(x)
    _check_weight(w1, "w1", K)
    _check_weight(w3, "w3", K)
    _check_mxfp4_buffer(w1, "w1")
    _check_mxfp4_buffer(w3, "w3")
    N = w1.rows
    if w3.rows != N:
        raise ValueError(f"w1 has {N} rows, w3 {w3.rows}")
    for name, t in (("gate_add", gate_add), ("up_add", up_add)):
        if t is not None:
            _check_device_tensor(t, name, torch.float32)
            if tuple(t.shape) != (M, N):
                raise ValueError(f"{name} must have shape ({M}, {N})")
    if quantize:
        if out is not None or out_dtype is not None:
            raise ValueError("quantize=True makes its own Mx8Tensor: out and out_dtype do not apply")
        if N % 256:
            raise ValueError(f"quantize=True needs N to be a multiple of 256, got {N}")
        flags = _lib.OUT_MXINT8
    else:
        dtype = _check_out(out, out_dtype, (M, N))
        flags = _lib.OUT_F32 if dtype == torch.float32 else 0
    _same_device(device, w1=w1.buf, w3=w3.buf, gate_add=gate_add, up_add=up_add, out=out)
    with _lib.on_device(device, stream):
        if quantize:
            res = Mx8Tensor(torch.empty(_mxint8_bytes(M, N), dtype=torch.uint8, device=device), M, N)
            out = res.buf
        else:
            out = res = torch.empty((M, N), dtype=dtype, device=device) if out is None else out
        ws, wp, wn = _workspace(M, N, K, x_type, device)
        rc = _lib.lib().qmlp_w4a8_swiglu(xp, x_type, stride, w1.buf.data_ptr(), w3.buf.data_ptr(),
                                         None if gate_add is None else gate_add.data_ptr(),
                                         None if up_add is None else up_add.data_ptr(), out.data_ptr(), wp, wn, M, N, K,
                                         flags, _lib.device_stream(device, stream))
        _lib.check(rc, "w4a8_swiglu")
    return res


def w4a8_mlp(x, weights, residual=None, out=None, out_dtype=None, adapters=None, plan=None, rows=None, stream=None):
    """``out = residual + down(silu(gate(x)) * up(x))`` with 8-bit activations and mxfp4 ``MLPWeights``.

    ``x`` as in ``w4a8_linear``, ``residual`` / ``out`` / ``out_dtype`` as its.  ``adapters`` (``MLPAdapters``) and the
    batch's ``plan``: low-rank adapters beside the projections; those of gate and up read ``x`` as rows (``rows`` where
    ``x`` is an ``Mx8Tensor``), those of down the bf16 rows between the projections, which then are what the down
    projection quantises, for every token of the call: one without an adapter gets 8-bit values rounded twice, which
    differ by at most a step from those of a call without adapters of down, quantised from fp32.
    """
    if weights.fmt != "mxfp4":
        raise ValueError(f"8-bit activations need mxfp4 weights, got {weights.fmt}")
    gate_add = up_add = None
    w2 = None
    if adapters is not None:
        if plan is None:
            raise ValueError("adapters need the batch's plan (lora_plan)")
        if rows is None and not isinstance(x, Mx8Tensor):
            rows = x
        for name, stack, n, k in (("w1", adapters.w1, weights.intermediate, weights.hidden),
                                  ("w3", adapters.w3, weights.intermediate, weights.hidden),
                                  ("w2", adapters.w2, weights.hidden, weights.intermediate)):
            if stack is not None and (stack.n, stack.k) != (n, k):
                raise ValueError(f"adapters.{name} is for [{stack.n}, {stack.k}], the projection is [{n}, {k}]")
        if rows is None and (adapters.w1 is not None or adapters.w3 is not None):
            raise ValueError("rows must hold the block's input where x is an Mx8Tensor")
        if adapters.w1 is not None:
            gate_add = lora_linear(rows, adapters.w1, plan, out_dtype=torch.float32, stream=stream)
        if adapters.w3 is not None:
            up_add = lora_linear(rows, adapters.w3, plan, out_dtype=torch.float32, stream=stream)
        w2 = adapters.w2
    elif plan is not None or rows is not None:
        raise ValueError("plan and rows belong to adapters")
    if residual is not None and tuple(residual.shape) != (x.shape[0], weights.hidden):
        raise ValueError(f"residual must have shape ({x.shape[0]}, {weights.hidden})")
    if w2 is None:
        h = w4a8_swiglu(x, weights.w1, weights.w3, gate_add, up_add, quantize=True, stream=stream)
    else:
        h = w4a8_swiglu(x, weights.w1, weights.w3, gate_add, up_add, stream=stream)
        residual = lora_linear(h, w2, plan, base=residual, out_dtype=torch.float32, stream=stream)
    return w4a8_linear(h, weights.w2, residual=residual, out=out, out_dtype=out_dtype, stream=stream)
