"""Low-rank adapters on the GPU against the formula in 64 bits.

The bound of an output's error: t = A x is a sum of exact products (16-bit operands) that the matrix cores
take in steps of 32, each rounding at most twice, then over 8 waves and at most 32 pieces: (2 K / 32 + 50) 2^-23 of
the summed magnitudes.  The scale rounds it once more, its split into three 16-bit parts loses at most 2^-24 of it
(bf16) or of the token's largest (fp16).  B t: two products for each 16 ranks, each rounding at most twice, 2^-23
of the summed magnitudes.  The base's addition and an output's own rounding come on top."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _np(t):
    return t.double().cpu().numpy()


def _adapters(ranks, N, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [((torch.randn(r, K, generator=g) * K ** -0.5).to(dtype), (torch.randn(N, r, generator=g) * 0.3).to(dtype),
             (-1) ** i * (0.5 + i)) for i, r in enumerate(ranks)]


def _oracle(x, adapters, ids):
    """The adapters' part of the outputs and what bounds its rounding, in float64."""
    M, K = x.shape
    N = adapters[0][1].shape[0]
    y, err = np.zeros((M, N)), np.zeros((M, N))
    for i, (a, b, s) in enumerate(adapters):
        rows = np.nonzero(ids == i)[0]
        if not len(rows):
            continue
        s = float(np.float32(s))
        a, b, v = _np(a), _np(b), x[rows]
        t = v @ a.T * s
        et = (2 * K / 32 + 50) * 2.0 ** -23 * (np.abs(v) @ np.abs(a).T) * abs(s) + 2.0 ** -23 * np.abs(t)
        et += 2.0 ** -24 * np.abs(t).max(axis=1, keepdims=True)
        units = -(-a.shape[0] // 16)
        y[rows] = t @ b.T
        err[rows] = et @ np.abs(b).T + 4 * units * 2.0 ** -23 * ((np.abs(t) + et) @ np.abs(b).T)
    return y, err


def _check(pkg, cuda, ids, ranks, N, K, dtype, seed=0, stride=0):
    M = len(ids)
    g = torch.Generator().manual_seed(seed + M)
    x = torch.randn(M, K + stride, generator=g).to(dtype)[:, :K]
    adapters = _adapters(ranks, N, K, dtype, seed)
    y, err = _oracle(_np(x), adapters, np.asarray(ids))
    stack = pkg.pack_lora([(a.to(cuda), b.to(cuda), s) for a, b, s in adapters])
    plan = pkg.lora_plan(torch.tensor(ids, dtype=torch.int32, device=cuda), len(ranks))
    x = x.to(cuda) if not stride else torch.cat([x, x], dim=1).to(cuda)[:, :K]
    got = pkg.lora_linear(x, stack, plan, out_dtype=torch.float32)
    assert got.shape == (M, N)
    worst = np.abs(_np(got) - y) - err
    assert (worst <= 0).all(), (worst.max(), np.unravel_index(worst.argmax(), worst.shape))
    gotb = pkg.lora_linear(x, stack, plan)
    assert torch.equal(gotb, got.bfloat16())
    for bd in (torch.bfloat16, torch.float32):
        base = torch.randn(M, N, generator=g).to(bd).to(cuda)
        full = y + _np(base)
        f32 = pkg.lora_linear(x, stack, plan, base=base, out_dtype=torch.float32)
        assert (np.abs(_np(f32) - full) <= err + 2.0 ** -24 * (np.abs(full) + err)).all()
        b16 = pkg.lora_linear(x, stack, plan, base=base)
        assert torch.equal(b16, f32.bfloat16())
        keep = base.clone()
        assert pkg.lora_linear(x, stack, plan, base=keep, out=keep) is keep
        assert torch.equal(keep, b16 if bd == torch.bfloat16 else f32)
        without = torch.tensor([not 0 <= i < len(ranks) for i in ids])
        assert torch.equal(f32[without.to(cuda)], base[without.to(cuda)].float())
    return x, stack, plan, got


CASES = [  # ids, ranks, N, K
    ([0], [1], 1, 32), ([0], [16], 5120, 5120), ([2], [8, 16, 4], 64, 17408), ([-1], [16], 72, 64),
    ([0, 1, 2, 1, 0], [16, 3, 24], 136, 96), ([3, 7, -5, 1 << 30, 0, 0], [5] * 4, 65, 288), ([0] * 16, [16], 128, 512),
    ([0] * 17, [32], 200, 1056), (list(range(32)), [(7 * i) % 64 + 1 for i in range(32)], 1000, 2080),
    (list(range(40, -24, -1)), [16] * 41, 96, 544), ([0] * 64, [128], 63, 320), ([0] * 65, [128], 64, 320),
    ([i % 3 for i in range(85)], [24] * 3, 257, 5120), ([i // 17 - 1 for i in range(85)], [24] * 3, 5121, 320),
    ([0] * 127, [1], 8, 32), ([i % 130 for i in range(200)], [17] * 130, 33, 64), ([0] * 300, [64, 64], 640, 2048),
    ([(i * i) % 9 - 1 for i in range(777)], [64, 33, 1, 128, 16, 15, 40, 100], 1032, 544),
    ([i // 700 for i in range(2000)], [48, 16, 80], 264, 1024), ([-1] * 100, [16], 56, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_lora_linear(pkg, cuda, case, dtype):
    ids, ranks, N, K = CASES[case]
    print(f"case lora {len(ids)} tokens, {len(ranks)} adapters, {N}x{K} {dtype}", flush=True)
    _check(pkg, cuda, ids, ranks, N, K, dtype, seed=case)


@pytest.mark.parametrize("M,ranks,N,K", [(65536, [1 + 3 * i % 20 for i in range(1024)], 40, 64), (65536, [33], 9, 32),
                                         (3, [4, 130 - 2], 1 << 20, 32), (2, [20], 5, 1 << 20), (65, [20, 7], 5, 1 << 20)])
def test_largest_sizes(pkg, cuda, M, ranks, N, K):
    """The most tokens with the most adapters and with one, the most features, the longest rows."""
    print(f"case lora {M}x{N}x{K}, {len(ranks)} adapters", flush=True)
    ids = torch.randint(-1, len(ranks) + 1, (M,), generator=torch.Generator().manual_seed(N)).tolist()
    _check(pkg, cuda, ids, ranks, N, K, torch.bfloat16, seed=3)


def test_strided_rows(pkg, cuda):
    for M in (3, 70):
        _check(pkg, cuda, [i % 2 for i in range(M)], [20, 7], 100, 96, torch.bfloat16, stride=96)


def test_the_order_of_the_tokens_changes_no_bit(pkg, cuda):
    M, L, N, K = 150, 5, 320, 1056
    adapters = [(a.to(cuda), b.to(cuda), s) for a, b, s in _adapters([16, 40, 8, 16, 3], N, K, torch.bfloat16, 3)]
    stack = pkg.pack_lora(adapters)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(M, K, generator=g).bfloat16().to(cuda)
    ids = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32).to(cuda)
    y = pkg.lora_linear(x, stack, pkg.lora_plan(ids, L), out_dtype=torch.float32)
    for _ in range(3):
        p = torch.randperm(M, generator=g).to(cuda)
        z = pkg.lora_linear(x[p].contiguous(), stack, pkg.lora_plan(ids[p].contiguous(), L), out_dtype=torch.float32)
        assert torch.equal(z, y[p])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_that_are_not_numbers_stay_apart(pkg, cuda, dtype):
    for M in (5, 90):
        adapters = [(a.to(cuda), b.to(cuda), s) for a, b, s in _adapters([16, 4], 72, 64, dtype, 3)]
        stack = pkg.pack_lora(adapters)
        x = torch.randn(M, 64, generator=torch.Generator().manual_seed(M)).to(dtype).to(cuda)
        plan = pkg.lora_plan(torch.tensor([i % 2 for i in range(M)], dtype=torch.int32, device=cuda), 2)
        clean = pkg.lora_linear(x, stack, plan)
        x[1, 5], x[2, 63] = float("nan"), float("inf")
        y = pkg.lora_linear(x, stack, plan)
        ok = torch.ones(M, dtype=torch.bool, device=cuda)
        ok[[1, 2]] = False
        assert torch.equal(y[ok], clean[ok]) and y[1].isnan().all()
        # an infinity stays what the formula makes of it: t infinite, y by the signs of t and b
        a, b, s = (v if isinstance(v, float) else _np(v) for v in adapters[0])
        with np.errstate(invalid="ignore"):
            want = (s * _np(x)[2:3] @ a.T) @ b.T
        got = _np(y)[2:3]
        assert (np.isnan(want) == np.isnan(got)).all() and np.array_equal(want[~np.isnan(want)], got[~np.isnan(want)])


@pytest.mark.parametrize("scale", [2.0 ** -24, 2.0 ** -12, 1.0, 2.0 ** 6])
def test_small_and_large_fp16_sums(pkg, cuda, scale):
    """fp16 adapters: sums far outside fp16's normal range keep their bits."""
    M, N, K = 20, 40, 64
    adapters = [(a, b, s * scale * 2.0 ** 10) for a, b, s in _adapters([16, 9], N, K, torch.float16, 5)]
    ids = np.array([i % 2 for i in range(M)])
    x = (torch.randn(M, K, generator=torch.Generator().manual_seed(4)) * 300).half()
    y, err = _oracle(_np(x), adapters, ids)
    stack = pkg.pack_lora([(a.to(cuda), b.to(cuda), s) for a, b, s in adapters])
    got = pkg.lora_linear(x.to(cuda), stack, pkg.lora_plan(torch.tensor(ids, dtype=torch.int32, device=cuda), 2),
                          out_dtype=torch.float32)
    assert (np.abs(_np(got) - y) <= err).all()


@pytest.mark.parametrize("run", [0, 1, 63, 64, 100, 700, 65536])
def test_plan_groups_every_token_once(pkg, cuda, run):
    """Tokens in any order (0) and in runs of one adapter."""
    for M, L in ((1, 1), (16, 3), (64, 1024), (65, 1), (700, 37), (65536, 1024)):
        g = torch.Generator().manual_seed(M)
        ids = torch.randint(-2, L + 2, (M,), generator=g, dtype=torch.int32)
        if run:
            ids = ids.repeat_interleave(run)[:M].contiguous()
        plan = pkg.lora_plan(ids.to(cuda), L)
        w = plan.buf.cpu().numpy()
        T = 16 if M <= 64 else 32
        most = M // T + min(M, L + 1)
        tiles = w[4:4 + 4 * w[3]].reshape(-1, 4)
        order = w[4 + 4 * most:]
        assert w[1] == M and w[2] == L and w[3] <= most and len(order) == M
        assert np.array_equal(np.sort(order), np.arange(M))
        at = 0
        for adapter, first, rows, _ in tiles:
            assert first == at and 1 <= rows <= T
            mine = ids.numpy()[order[first:first + rows]]
            assert (mine == adapter).all() if adapter >= 0 else ((mine < 0) | (mine >= L)).all()
            at += rows
        assert at == M


def test_offsets_beyond_32_bits(pkg, cuda):
    """An output of more than 2^32 values and rows of x more than 2^32 bytes apart: the last rows, against the same
    rows by themselves."""
    M, N, K = 40000, 120000, 64
    g = torch.Generator(device=cuda).manual_seed(1)
    stack = pkg.pack_lora([(torch.randn(16, K, generator=g, device=cuda).bfloat16(),
                            torch.randn(N, 16, generator=g, device=cuda).bfloat16(), 0.5) for _ in range(2)])
    stride = 60000
    x = torch.randn(M * stride, generator=g, device=cuda, dtype=torch.bfloat16).view(M, stride)[:, :K]
    ids = (torch.arange(M, device=cuda) % 3).to(torch.int32)
    y = pkg.lora_linear(x, stack, pkg.lora_plan(ids, 2))
    for rows in (slice(0, 70), slice(M - 70, M)):
        few = pkg.lora_linear(x[rows].contiguous(), stack, pkg.lora_plan(ids[rows].contiguous(), 2))
        assert torch.equal(y[rows], few) and few.abs().max() > 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [6, 70])
def test_sums_next_to_the_largest_number(pkg, cuda, M, dtype):
    """Scaled sums up to fp32's largest number, where a rounding to bf16 (from 2^128 - 2^119 on) would be an infinity,
    give finite outputs.  t is one value of x in its first rank, so that the scaled sum is the scale with a sign."""
    K, N, most = 32, 24, float(np.finfo(np.float32).max)
    edge = 2.0 ** 128 - 2.0 ** 119  # half way from bf16's largest number to the infinity
    scales = [edge * (1 - 2.0 ** -24), edge, edge * (1 + 2.0 ** -23), most, -most, 3.4e38]
    g = torch.Generator().manual_seed(M)
    adapters = []
    for s in scales:
        a = torch.zeros(3, K)
        a[0, 0], a[1, 1] = 1.0, 2.0 ** -14
        adapters.append((a.to(dtype), (torch.rand(N, 3, generator=g) * 1.5 - 0.75).to(dtype), s))
    x = torch.ones(M, K)
    x[::2] = -1.0
    x = x.to(dtype)
    ids = np.arange(M) % len(scales)
    y, err = _oracle(_np(x), adapters, ids)
    stack = pkg.pack_lora([(a.to(cuda), b.to(cuda), s) for a, b, s in adapters])
    got = pkg.lora_linear(x.to(cuda), stack, pkg.lora_plan(torch.tensor(ids, dtype=torch.int32, device=cuda), len(scales)),
                          out_dtype=torch.float32)
    assert np.isfinite(y).all() and torch.isfinite(got).all()
    assert (np.abs(_np(got) - y) <= err).all()
