"""Low-rank adapters of many requests at once, beside a shared projection.

* ``pack_lora([(a, b, scale), ...])`` -> ``LoraStack``: the adapters of one projection, laid out once when they
  are loaded (``a`` ``[rank, K]``, ``b`` ``[N, rank]``, both bf16 or both fp16; ranks from 1 to 128 may differ);
* ``lora_plan(ids, adapters)`` -> ``LoraPlan``: which tokens share an adapter, made once for a batch and used by
  every projection of every layer; ``ids`` int32 ``[M]``, the adapter of each token (any other number: none);
* ``lora_linear(x, stack, plan, base=...)``: ``out[m] = base[m] + scale_a b_a (a_a x[m])``.

``base`` may be the shared projection's output, or what the projection adds itself: with an fp32 ``out`` the
result is the ``residual`` of ``w4a8_linear`` and ``mxfp4_linear``, and ``gate_add`` / ``up_add`` of
``w4a8_swiglu``, so that the sum of both is rounded once.  Sums are fp32.  Sizes: any M up to 65536, any N, K a
multiple of 32, up to 1024 adapters.  The reference's projections have no adapters
(``docker/qwen-c2-graft/graft/mlp.py:402-423``).

Every call runs on the inputs' GPU, on ``stream`` or that GPU's current stream, may be captured into a HIP
graph (``pack_lora`` reads its scales from the host and may not) and allocates its output and scratch memory from
torch's caching allocator there.  A replayed graph with ``lora_plan`` in it follows new ids.  Errors:
``ValueError`` for wrong shapes, dtypes or devices, ``QmlpError`` for launch failures.
"""
import functools
import struct
from dataclasses import dataclass

import torch

from . import _lib
from .mlp import _check_device_tensor, _same_device
from .mxfp4 import _check_out, _check_rows

MAX_RANK = 128
MAX_ADAPTERS = 1024


@dataclass(frozen=True)
class LoraStack:
    """The adapters of one projection in the kernels' layout."""

    a: torch.Tensor     # [rank units, K / 32, 64, 8], all adapters in turn
    b: torch.Tensor     # flat, per adapter [N / 64, rank / 32, 4, 64, 8]
    meta: torch.Tensor  # int32 [adapters, 4]: rank, rank units before, scale's bits, 32s of ranks before
    ranks: tuple
    max_rank: int
    adapters: int
    n: int
    k: int

    @property
    def device(self):
        return self.a.device

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.a, self.b, self.meta))


@dataclass(frozen=True)
class MLPAdapters:
    """The adapters of one feed-forward block, None where a projection has none; fields as in ``MLPWeights``."""

    w1: LoraStack = None  # gate_proj
    w2: LoraStack = None  # down_proj
    w3: LoraStack = None  # up_proj


@dataclass(frozen=True)
class LoraPlan:
    """A batch's tokens grouped by adapter."""

    buf: torch.Tensor  # int32, qmlp_lora_plan_bytes(tokens, adapters) bytes
    tokens: int
    adapters: int


def _units(ranks, size):
    """Units of ``size`` ranks of each adapter, and of those before it."""
    units = [-(-r // size) for r in ranks]
    return units, [sum(units[:i]) for i in range(len(units))]


def _scale_bits(scale, i):
    """The bits of adapter ``i``'s scale in fp32, where it has to be a finite number."""
    try:
        value = float(scale)
        packed = struct.pack("<f", value)
    except OverflowError:  # an integer beyond any float; a finite number beyond fp32
        value = float("inf")
    if not abs(value) < float("inf"):
        raise ValueError(f"adapter {i}: the scale must be finite in fp32, got {scale}")
    return struct.unpack("<i", packed)[0]


def pack_lora(adapters, stream=None):
    """``[(a [rank, K], b [N, rank], scale), ...]`` (GPU tensors, a number) -> ``LoraStack``.  ``scale`` is what the
    adapter's product is multiplied by (``alpha / rank`` as a rule), rounded to fp32."""
    adapters = list(adapters)
    if not 1 <= len(adapters) <= MAX_ADAPTERS:
        raise ValueError(f"need 1 to {MAX_ADAPTERS} adapters, got {len(adapters)}")
    first, bits = adapters[0][0], []
    for i, (a, b, scale) in enumerate(adapters):
        for name, t in (("a", a), ("b", b)):
            _check_device_tensor(t, f"adapter {i}: {name}")
            if t.dtype not in (torch.bfloat16, torch.float16) or t.dtype != first.dtype:
                raise ValueError(f"adapter {i}: {name} must be bf16 or fp16, all adapters alike, got {t.dtype}")
            if t.dim() != 2:
                raise ValueError(f"adapter {i}: {name} must be 2-D")
            if t.device != first.device:
                raise ValueError(f"adapter {i}: {name} is on {t.device}, the first adapter on {first.device}")
        rank, K = a.shape
        if not 1 <= rank <= MAX_RANK or b.shape[1] != rank:
            raise ValueError(f"adapter {i}: a is {tuple(a.shape)}, b {tuple(b.shape)}: ranks from 1 to {MAX_RANK}, alike")
        if K != first.shape[1] or b.shape[0] != adapters[0][1].shape[0]:
            raise ValueError(f"adapter {i}: a is {tuple(a.shape)}, b {tuple(b.shape)}, the first ones are "
                             f"{tuple(first.shape)} and {tuple(adapters[0][1].shape)}")
        if K == 0 or K % 32 or b.shape[0] == 0:
            raise ValueError(f"a must have a multiple of 32 columns and b rows, got {K} and {b.shape[0]}")
        bits.append(_scale_bits(scale, i))
    N, K = adapters[0][1].shape[0], first.shape[1]
    blocks = -(-N // 64)
    ranks = tuple(a.shape[0] for a, _, _ in adapters)
    units, before = _units(ranks, 16)
    units32, before32 = _units(ranks, 32)
    with _lib.on_device(first.device, stream):
        pa = torch.zeros((sum(units) * 16, K), dtype=first.dtype, device=first.device)
        pb = torch.empty((sum(units32), 32 * blocks * 64), dtype=first.dtype, device=first.device)
        for i, (a, b, _) in enumerate(adapters):
            pa[16 * before[i]:16 * before[i] + ranks[i]] = a
            wide = torch.zeros((blocks * 64, 32 * units32[i]), dtype=first.dtype, device=first.device)
            wide[:N, :ranks[i]] = b
            # feature 16 f + e of a block, rank 32 u + 8 h + j -> [block][u][f][lane 16 h + e][j]
            wide = wide.reshape(blocks, 4, 16, units32[i], 4, 8).permute(0, 3, 1, 4, 2, 5)
            pb[before32[i]:before32[i] + units32[i]] = wide.reshape(units32[i], -1)
        pa = pa.reshape(sum(units), 16, K // 32, 4, 8).permute(0, 2, 3, 1, 4).contiguous()
        meta = torch.tensor(list(zip(ranks, before, bits, before32)), dtype=torch.int32).to(first.device)
    return LoraStack(pa, pb, meta, ranks, max(ranks), len(ranks), N, K)


@functools.lru_cache(maxsize=4096)
def _plan_bytes(M, adapters):
    return _lib.lib().qmlp_lora_plan_bytes(M, adapters)


def lora_plan(ids, adapters, stream=None):
    """``ids`` int32 ``[M]`` on the GPU and the number of adapters that they name -> ``LoraPlan``."""
    _check_device_tensor(ids, "ids", torch.int32)
    if ids.dim() != 1 or not 1 <= ids.shape[0] <= 65536:
        raise ValueError(f"ids must hold 1 to 65536 tokens, got {tuple(ids.shape)}")
    if not 1 <= adapters <= MAX_ADAPTERS:
        raise ValueError(f"need 1 to {MAX_ADAPTERS} adapters, got {adapters}")
    M, device = ids.shape[0], ids.device
    nbytes = _plan_bytes(M, adapters)
    with _lib.on_device(device, stream):
        buf = torch.empty(nbytes // 4, dtype=torch.int32, device=device)
        _lib.check(_lib.lib().qmlp_lora_plan(ids.data_ptr(), M, adapters, buf.data_ptr(), nbytes,
                                             _lib.device_stream(device, stream)), "lora_plan")
    return LoraPlan(buf, M, adapters)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(M, K, max_rank):
    return _lib.lib().qmlp_lora_workspace_bytes(M, K, max_rank)


def lora_linear(x, stack, plan, base=None, out=None, out_dtype=None, stream=None):
    """``out[m] = base[m] + scale_a b_a (a_a x[m])`` for the adapter ``a`` of each token.

    ``x``: bf16 or fp16 ``[M, K]`` of the adapters' dtype, rows may be strided; ``base`` bf16 or fp32 ``[M, N]`` or
    None (zeros); ``out`` (or ``out_dtype`` when ``out`` is None) bf16, rounded once to nearest-even, or fp32.
    ``out`` may be the base itself.
    """
    if not isinstance(stack, LoraStack) or not isinstance(plan, LoraPlan):
        raise ValueError("stack must be a LoraStack (pack_lora) and plan a LoraPlan (lora_plan)")
    x_type, stride = _check_rows(x)
    M, K = x.shape
    N = stack.n
    if x.dtype != stack.a.dtype:
        raise ValueError(f"x is {x.dtype}, the adapters {stack.a.dtype}")
    if K != stack.k:
        raise ValueError(f"x has {K} columns, the adapters {stack.k}")
    if plan.tokens != M or plan.adapters != stack.adapters:
        raise ValueError(f"the plan is for {plan.tokens} tokens and {plan.adapters} adapters, x has {M} rows and the "
                         f"stack {stack.adapters} adapters")
    dtype = _check_out(out, out_dtype, (M, N))
    flags = _lib.OUT_F32 if dtype == torch.float32 else 0
    if base is not None:
        _check_device_tensor(base, "base")
        if base.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("base must be bf16 or fp32")
        if tuple(base.shape) != (M, N):
            raise ValueError(f"base must have shape ({M}, {N})")
        if base.dtype == torch.float32:
            flags |= _lib.RESIDUAL_F32
    device = x.device
    _same_device(device, stack=stack.a, plan=plan.buf, base=base, out=out)
    with _lib.on_device(device, stream):
        if out is None:
            out = x.new_empty((M, N), dtype=dtype)
        nbytes = _workspace_bytes(M, K, stack.max_rank)
        ws = x.new_empty(nbytes, dtype=torch.uint8)
        rc = _lib.lib().qmlp_lora_linear(x.data_ptr(), x_type, stride, stack.a.data_ptr(), stack.b.data_ptr(),
                                         stack.meta.data_ptr(), stack.adapters, stack.max_rank, plan.buf.data_ptr(),
                                         None if base is None else base.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                         nbytes, M, N, K, flags, _lib.device_stream(device, stream))
        _lib.check(rc, "lora_linear")
    return out
