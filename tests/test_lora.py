"""Low-rank adapters without a GPU: sizes and refusals of the entry points."""
import ctypes

import pytest
import torch

E_SHAPE, E_ALIGN, E_FORMAT, E_WORKSPACE, E_NULL = -1, -2, -3, -5, -6


def P(at):
    return ctypes.c_void_p(at)


X, A, B, META, PLAN, BASE, OUT, WS = (P(1 << k) for k in range(32, 40))

# (ids, ranks, N, K): sizes that together take every kernel that lora_linear launches, with A x in one piece of K, in
# several, and in fewer than K has because many adapters are loaded
FOUR = [i // 130 for i in range(520)]  # four requests
PATHS = [
    ([0, 1, 2], [128, 70, 16], 136, 5120), ([0] * 40, [32], 72, 8192), ([i % 3 for i in range(33)], [64, 40, 1], 65, 2048),
    (list(range(64)), [16] * 64, 33, 8192), ([5, 0], [8] * 6, 40, 17408), ([1, 1, -1, 0], [1, 9], 23, 512),
    ([4, 0], [8] * 5, 40, 5120), ([0, 1], [30, 20], 24, 2048), ([0, 1, 0], [30, 20], 25, 1024), ([2, 1, 0], [64, 50, 3], 48, 512),
    ([0] * 9, [40], 49, 544), ([1, 0, 0], [128, 65], 16, 288), ([0] * 64, [96], 17, 320),
    ([i % 2 for i in range(65)], [16, 5], 64, 1056), ([i % 2 for i in range(100)], [128, 5], 39, 2048),
    (FOUR, [17] * 60, 40, 4096), (FOUR, [64] * 4, 72, 4096), (FOUR, [1 + i % 16 for i in range(120)], 41, 4096),
    (FOUR, [33] * 300, 24, 4096), (FOUR, [2] * 109 + [128], 40, 2560),
]


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


def _path(pkg, M, N, K, L, rank, cus=256):
    out = (ctypes.c_int * 5)()
    assert pkg.lib().qmlp_lora_path(M, N, K, L, rank, cus, out) == 0
    return tuple(out)


def test_sizes_reach_every_kernel(pkg):
    """What the tests on the GPU run, both types each: every kernel of one launch and of two, with rows that a vector
    store fits and others, with K in one piece, in several, and in fewer because many adapters are loaded."""
    one, down, up, pieces = set(), set(), set(), set()
    for ids, ranks, N, K in PATHS:
        launches, tile, units, n, most = _path(pkg, len(ids), N, K, len(ranks), max(ranks))
        if launches == 1:
            one.add((units, N % 8 == 0))
        else:
            down.add((tile, units))
            up.add(N % 8 == 0)
            pieces.add((tile, n, most))
    assert one == {(u, w) for u in (1, 2, 4, 8) for w in (True, False)}
    assert down == {(t, u) for t in (1, 2) for u in (1, 2, 4, 8)} and up == {True, False}
    assert {(2, n, 8) for n in (8, 4, 2, 1)} <= pieces and {(1, 8, 8), (1, 4, 8)} <= pieces  # from eight pieces on
    assert any(most % 2 and n == most for _, n, most in pieces) and any(most % 2 and n < most for _, n, most in pieces)


def test_paths_are_within_the_kernels_limits(pkg):
    for K in (32, 512, 544, 5120, 17408, 1 << 20):
        for rank in (1, 16, 17, 33, 65, 128):
            for M in (1, 16, 17, 64, 65, 520, 2048, 65536):
                for L in (1, 60, 300, 1024):
                    launches, tile, units, n, most = _path(pkg, M, 64, K, L, rank)
                    assert tile == (1 if M <= 64 else 2) and 16 * units >= rank and units <= max(1, rank // 8)
                    assert 1 <= n <= most <= 8 and (launches == 2 or (tile == 1 and n == 1))
                    assert launches == 1 or n * -(-rank // 16) * 16 * 4 * M <= pkg.lib().qmlp_lora_workspace_bytes(M, K, rank)
    out = (ctypes.c_int * 5)()
    for bad in ((0, 64, 64, 1, 1, 256), (65537, 64, 64, 1, 1, 256), (1, 0, 64, 1, 1, 256), (1, 64, 48, 1, 1, 256),
                (1, 64, 64, 0, 1, 256), (1, 64, 64, 1025, 1, 256), (1, 64, 64, 1, 129, 256), (1, 64, 64, 1, 1, 0)):
        assert pkg.lib().qmlp_lora_path(*bad, out) == E_SHAPE
    assert pkg.lib().qmlp_lora_path(1, 64, 64, 1, 1, 256, None) == E_NULL


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
