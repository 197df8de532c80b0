"""Low-rank adapters without a GPU: sizes and refusals of the entry points."""
import ctypes

import pytest
import torch

E_SHAPE, E_ALIGN, E_FORMAT, E_WORKSPACE, E_NULL = -1, -2, -3, -5, -6


def P(at):
    return ctypes.c_void_p(at)


X, A, B, META, PLAN, BASE, OUT, WS = (P(1 << k) for k in range(32, 40))


def test_sizes(pkg):
    lib = pkg.lib()
    for M, L in ((1, 1), (16, 3), (64, 1024), (65, 1), (700, 37), (65536, 1024)):
        T = 16 if M <= 64 else 32
        assert lib.qmlp_lora_plan_bytes(M, L) == 4 * (4 + 4 * (M // T + min(M, L + 1)) + M)
    for bad in ((0, 1), (65537, 1), (1, 0), (1, 1025), (-1, 4)):
        assert lib.qmlp_lora_plan_bytes(*bad) == 0
    Ms = list(range(1, 300)) + [1023, 1024, 65535, 65536]
    for K in (32, 544, 17408, 1 << 20):
        for rank in (1, 16, 17, 128):
            sizes = [lib.qmlp_lora_workspace_bytes(M, K, rank) for M in Ms]
            assert sizes[0] > 0 and sizes == sorted(sizes)
            assert sizes[-1] >= 65536 * -(-rank // 16) * 16 * 4
    for bad in ((0, 32, 1), (65537, 32, 1), (1, 48, 1), (1, 0, 1), (1, 32, 0), (1, 32, 129)):
        assert lib.qmlp_lora_workspace_bytes(*bad) == 0


def test_plan_refusals(pkg):
    lib = pkg.lib()
    n = lib.qmlp_lora_plan_bytes(40, 3)

    def f(ids=X, M=40, L=3, plan=PLAN, nb=n):
        return lib.qmlp_lora_plan(ids, M, L, plan, nb, None)

    assert f(ids=None) == E_NULL and f(plan=None) == E_NULL
    assert f(ids=P((1 << 32) + 2)) == E_ALIGN and f(plan=P((1 << 36) + 4)) == E_ALIGN
    for kw in ({"M": 0}, {"M": 65537}, {"L": 0}, {"L": 1025}, {"plan": P((1 << 32) + 16)}):
        assert f(**kw) == E_SHAPE, kw
    assert f(nb=n - 1) == E_WORKSPACE


def test_linear_refusals(pkg):
    lib = pkg.lib()

    def f(x=X, xt=0, xs=256, a=A, b=B, meta=META, L=3, rank=16, plan=PLAN, base=None, out=OUT, ws=WS, wsb=1 << 30, M=40,
          N=64, K=256, flags=0):
        return lib.qmlp_lora_linear(x, xt, xs, a, b, meta, L, rank, plan, base, out, ws, wsb, M, N, K, flags, None)

    for arg in ("x", "a", "b", "meta", "plan", "out", "ws"):
        assert f(**{arg: None}) == E_NULL, arg
    for arg in ("x", "a", "b", "meta", "plan", "base", "out", "ws"):
        assert f(**{arg: P((1 << 41) + 8)}) == E_ALIGN, arg
    assert f(xt=2) == E_FORMAT and f(xt=4) == E_FORMAT and f(flags=4) == E_FORMAT
    for kw in ({"M": 0}, {"M": 65537}, {"N": 0}, {"K": 48}, {"K": 0}, {"L": 0}, {"L": 1025}, {"rank": 0}, {"rank": 129},
               {"xs": 255}, {"xs": 260}, {"xs": 1 << 50}, {"N": 1 << 21}):
        assert f(**kw) == E_SHAPE, kw
    assert f(wsb=lib.qmlp_lora_workspace_bytes(40, 256, 16) - 1) == E_WORKSPACE
    for kw in ({"base": P((1 << 38) + 64)}, {"base": OUT, "flags": 1}, {"base": OUT, "flags": 2}, {"out": X}, {"out": PLAN},
               {"out": META}, {"out": A}, {"out": B}, {"ws": X}, {"ws": PLAN}, {"ws": META}, {"ws": A}, {"ws": B}, {"ws": OUT},
               {"ws": BASE, "base": BASE}):
        assert f(**kw) == E_SHAPE, kw


def test_python_refusals_need_no_gpu(pkg):
    a, b = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 4, dtype=torch.bfloat16)
    for bad in ([], [(a, b, 1.0)] * 1025):
        with pytest.raises(ValueError, match="1 to 1024"):
            pkg.pack_lora(bad)
    with pytest.raises(ValueError, match="GPU"):
        pkg.pack_lora([(a, b, 1.0)])
    with pytest.raises(ValueError, match="GPU"):
        pkg.lora_plan(torch.zeros(3, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="LoraStack"):
        pkg.lora_linear(a, None, None)


@pytest.fixture
def cpu_pack(pkg, monkeypatch):
    """``pack_lora`` without its test for GPU tensors: all it does besides is torch's own operations."""
    import contextlib

    from qwen_mlp_amd import _lib, lora

    monkeypatch.setattr(lora, "_check_device_tensor", lambda t, name: None)
    monkeypatch.setattr(_lib, "on_device", lambda device, stream=None: contextlib.nullcontext())
    return pkg.pack_lora


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan"), 1e39, -1e39, 2.0 ** 128 - 2.0 ** 103,
                                   pytest.param(10 ** 400, id="10**400")])
def test_scales_that_fp32_does_not_hold_are_refused(cpu_pack, scale):
    """The scale is kept in fp32: what is not a finite number there (from 2^128 - 2^103 on, half a step beyond the
    largest, a number becomes an infinity) is refused like any other bad argument."""
    a, b = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="adapter 1: the scale must be finite"):
        cpu_pack([(a, b, 1.0), (a, b, scale)])


def test_scales_are_rounded_to_fp32(cpu_pack):
    a, b = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 4, dtype=torch.bfloat16)
    most = torch.finfo(torch.float32).max
    scales = [0.1, most, -most, 2.0 ** 128 - 2.0 ** 103 - 2.0 ** 76, 2.0 ** -149, 0.0, 7, torch.tensor(0.3)]
    meta = cpu_pack([(a, b, s) for s in scales]).meta
    got = meta[:, 2].contiguous().view(torch.float32)
    assert torch.equal(got, torch.tensor([float(s) for s in scales], dtype=torch.float64).float())
    assert torch.isfinite(got).all()
