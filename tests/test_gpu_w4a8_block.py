"""The feed-forward block with 8-bit activations, the norm in front of it and adapters beside it: the calls of a
decoder layer's second half together, against the formulas in 64 bits, in graphs and on streams.

The bound of an output's error.  The gate's and up's sums: as the products' and the adapters' own tests derive
them, and one more rounding where both are added.  h = silu(g) u: as the gate/up pair's test derives it.  What the
block quantises is that h: where its error could change an integer or its block's scale, the reference allows what
either would give (``_either``), and the down product multiplies that by the weights' magnitudes."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as omx
from oracle import mxint8 as omi

pytestmark = pytest.mark.gpu
H, I = 512, 1280


def _np(t):
    return t.double().cpu().numpy()


def _state(cuda, seed=0):
    g = torch.Generator().manual_seed(seed)
    return {f"{n}.weight": (torch.randn(*s, generator=g) * 0.05).bfloat16().to(cuda)
            for n, s in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I)))}


def _adapters(pkg, cuda, seed, which=("w1", "w2", "w3"), L=3):
    g = torch.Generator().manual_seed(seed)
    raw, stacks = {}, {}
    for f in which:
        n, k = (H, I) if f == "w2" else (I, H)
        raw[f] = [((torch.randn(r, k, generator=g) * k ** -0.5).bfloat16(), (torch.randn(n, r, generator=g) * 0.2).bfloat16(),
                   0.5 + i) for i, r in enumerate((16, 5, 40)[:L])]
        stacks[f] = pkg.pack_lora([(a.to(cuda), b.to(cuda), s) for a, b, s in raw[f]])
    return raw, pkg.MLPAdapters(**stacks)


def _lora(x, ex, raw, ids):
    """The adapters' part for rows x (known to ex) and its bound (tests/test_gpu_lora.py)."""
    N = raw[0][1].shape[0]
    y, err = np.zeros((x.shape[0], N)), np.zeros((x.shape[0], N))
    for i, (a, b, s) in enumerate(raw):
        rows = ids == i
        if not rows.any():
            continue
        a, b, v, ev = _np(a), _np(b), x[rows], ex[rows]
        t, K = s * v @ a.T, x.shape[1]
        et = abs(s) * (((2 * K / 32 + 50) * 2.0 ** -23 * (np.abs(v) + ev) + ev) @ np.abs(a).T)
        et += 2.0 ** -23 * (np.abs(t) + et) + 2.0 ** -24 * (np.abs(t) + et).max(axis=1, keepdims=True)
        y[rows] = t @ b.T
        err[rows] = et @ np.abs(b).T + 4 * -(-a.shape[0] // 16) * 2.0 ** -23 * ((np.abs(t) + et) @ np.abs(b).T)
    return y, err


def _q8(x):
    return omi.dequantize(*omi.quantize(x))


def _either(h, e):
    """The most that quantising something within e of h can differ from quantising h: a block's scale is that of its
    largest possible or its smallest possible maximum, and rounding is monotonic."""
    mid = _q8(h)
    out = np.zeros_like(h)
    for top in (np.maximum(np.abs(h) - e, 0), np.abs(h) + e):
        top = top.reshape(h.shape[0], -1, 32).max(axis=2, keepdims=True)
        step = np.exp2(np.floor(np.log2(np.maximum(top, 2.0 ** -120))) - 6)
        for v in (h - e, h + e):
            q = np.rint(v.reshape(h.shape[0], -1, 32) / step).clip(-127, 127) * step
            out = np.maximum(out, np.abs(q.reshape(h.shape) - mid))
    return out


def _silu(g):
    return g / (1 + np.exp(-np.clip(g, -700, 700)))


def _sum_error(K, magnitudes):
    return (4 * (K / 64 + 1) + 32) * 2.0 ** -23 * magnitudes


def _block(sd, x, raw=None, ids=None):
    """The block's output for rows x (float64), without a residual, and the bound of its error."""
    w = {n: omx.dequantize(*omx.quantize(_np(sd[f"{n}.weight"]))) for n in ("gate_proj", "up_proj", "down_proj")}
    raw, v, parts = raw or {}, _q8(x), []
    for name, f in (("gate_proj", "w1"), ("up_proj", "w3")):
        y, mag = omx.linear(v, w[name])
        e = _sum_error(H, mag)
        if f in raw:
            d, ed = _lora(x, np.zeros_like(x), raw[f], ids)
            y, e = y + d, e + ed
            e = e + 2.0 ** -23 * (np.abs(y) + e)
        parts.append((y, e))
    (g, ge), (u, ue) = parts
    s = _silu(g)
    h = s * u
    eh = 1.1 * ge * (np.abs(u) + ue) + (np.abs(s) + 1.1 * ge) * ue + (8 + np.abs(g)) * 2.0 ** -23 * np.abs(h) + 1e-37
    d = ed = 0.0
    if "w2" in raw:  # h goes on as bf16 rows
        lo, mid, hi = (torch.from_numpy(t).bfloat16().double().numpy() for t in (h - eh, h, h + eh))
        h, eh = mid, np.maximum(hi - mid, mid - lo)
        d, ed = _lora(h, eh, raw["w2"], ids)
    either = _either(h, eh)
    y, mag = omx.linear(_q8(h), w["down_proj"])
    more = either @ np.abs(w["down_proj"]).T
    return y + d, _sum_error(I, mag + more) + more + ed + 2.0 ** -23 * np.abs(y + d)


def _normed(hd, w, eps=1e-6):
    return hd / np.sqrt((hd * hd).mean(axis=1, keepdims=True) + eps) * (1 + _np(w))


@pytest.mark.parametrize("M", [1, 3, 16, 30, 64, 85, 200])
@pytest.mark.parametrize("which", [(), ("w1",), ("w2",), ("w1", "w3"), ("w1", "w2", "w3")])
def test_block(pkg, cuda, M, which):
    print(f"case block {M} {which}", flush=True)
    sd = _state(cuda, M)
    mlp = pkg.Qwen36MLP(cuda, sd, weight_format="mxfp4", activation_format="mxint8", max_tokens=M)
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, H, generator=g).bfloat16()
    res = torch.randn(M, H, generator=g)
    ids = np.array([(i * 7) % 5 - 1 for i in range(M)])
    raw, ad = _adapters(pkg, cuda, M, which) if which else (None, None)
    kw = dict(adapters=ad, plan=pkg.lora_plan(torch.tensor(ids, dtype=torch.int32, device=cuda), 3)) if which else {}
    y, bound = _block(sd, _np(x), raw, ids)
    got = mlp.forward(x.to(cuda), residual=res.to(cuda), out_dtype=torch.float32, **kw)
    full = y + _np(res)
    # the residual is added once more, to the sum or to the adapters' part of it
    assert (np.abs(_np(got) - full) <= bound + 2.0 ** -23 * (np.abs(full) + np.abs(_np(res)) + bound)).all()
    # the pieces by themselves give the same bits, and so do other leading dimensions and a given output
    xg, rg = x.to(cuda), res.to(cuda)
    out = torch.empty(1, 1, M, H, device=cuda)
    assert mlp.forward(xg.view(1, 1, M, H), residual=rg.view(1, 1, M, H), out=out, **kw) is out
    assert torch.equal(out.view(M, H), got)
    assert torch.equal(mlp(xg, residual=rg, out=rg, **kw), got)
    b = mlp.forward(xg, residual=x.to(cuda), **kw)
    assert b.dtype == torch.bfloat16 and torch.equal(b, mlp.forward(xg, residual=x.to(cuda), out_dtype=torch.float32, **kw).bfloat16())


@pytest.mark.parametrize("M", [1, 16, 70])
def test_the_decoders_half_layer(pkg, cuda, M):
    """forward_add_rmsnorm is add_rmsnorm and the block, and forward_rmsnorm the same without an addition, with and
    without adapters, on bf16 and fp32 streams; other formats take the norm's rows."""
    sd = _state(cuda, 5)
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, H, generator=g).bfloat16().to(cuda), (torch.randn(H, generator=g) * 0.1).bfloat16().to(cuda)
    raw, ad = _adapters(pkg, cuda, 1)
    ids = torch.tensor([i % 4 - 1 for i in range(M)], dtype=torch.int32, device=cuda)
    kws = ({}, dict(adapters=ad, plan=pkg.lora_plan(ids, 3)))
    mlp = pkg.Qwen36MLP(cuda, sd, weight_format="mxfp4", activation_format="mxint8", max_tokens=M)
    for rt in (torch.bfloat16, torch.float32):
        r = torch.randn(M, H, generator=g).to(rt).to(cuda)
        for kw in kws:
            h, rows, n = pkg.add_rmsnorm(x, r, w, output="both")
            want = pkg.w4a8_mlp(n, mlp.weights, residual=h, out_dtype=rt, rows=rows if kw else None, **kw)
            got = mlp.forward_add_rmsnorm(x, r, w, out_dtype=rt, **kw)
            assert got.dtype == rt and torch.equal(got, want)
            assert torch.equal(mlp.forward(rows, residual=h, out_dtype=rt, **kw), want)
            inplace = r.clone().view(1, M, H)
            assert mlp.forward_add_rmsnorm(x.view(1, M, H), inplace, w, out=inplace, **kw) is inplace
            assert torch.equal(inplace.view(M, H), want)
            if rt == torch.bfloat16:
                assert torch.equal(mlp.forward_rmsnorm(h, w, **kw), want)
        hd = _np(h)
        y, bound = _block(sd, _np(rows), raw, ids.cpu().numpy())
        half_step = 2.0 ** -8 if rt == torch.bfloat16 else 2.0 ** -24
        bound = bound + 2.0 ** -23 * (np.abs(y + hd) + np.abs(hd) + bound)
        assert (np.abs(_np(want) - (y + hd)) <= bound + half_step * (np.abs(y + hd) + bound)).all()
        # the norm's fp32 error is below 2^-17 of the value, its rounding half a bf16 step
        normed = _normed(hd, w)
        assert (np.abs(_np(rows) - normed) <= (2.0 ** -17 + 2.0 ** -8 * (1 + 2.0 ** -17)) * np.abs(normed)).all()
        for fmt in ("bf16", "bfp8", "bf4", "mxfp4"):
            other = pkg.Qwen36MLP(cuda, sd, weight_format=fmt, max_tokens=M)
            want = other.forward(rows, residual=h.contiguous(), out_dtype=rt)
            assert torch.equal(other.forward_add_rmsnorm(x, r, w, out_dtype=rt), want)


def test_refusals(pkg, cuda):
    sd = _state(cuda)
    mlp = pkg.Qwen36MLP(cuda, sd, weight_format="mxfp4", activation_format="mxint8", max_tokens=4)
    a4 = pkg.Qwen36MLP(cuda, sd, weight_format="mxfp4", max_tokens=4)
    assert a4.activation_format == "mxfp4" and mlp.activation_format == "mxint8"
    _, ad = _adapters(pkg, cuda, 1)
    x = torch.zeros(4, H, dtype=torch.bfloat16, device=cuda)
    w = x[0].clone()
    plan = pkg.lora_plan(torch.zeros(4, dtype=torch.int32, device=cuda), 3)
    for fmt, act in (("bfp8", "mxint8"), ("bf16", "mxfp4"), ("mxfp4", "int8")):
        with pytest.raises(ValueError, match="activation format"):
            pkg.Qwen36MLP(cuda, sd, weight_format=fmt, activation_format=act, max_tokens=4)
    for call in (lambda: a4.forward(x, adapters=ad, plan=plan), lambda: a4.forward_rmsnorm(x, w, plan=plan),
                 lambda: a4.forward_add_rmsnorm(x, x, w, adapters=ad, plan=plan)):
        with pytest.raises(ValueError, match="mxint8"):
            call()
    bad = [lambda: mlp.forward(x, adapters=ad), lambda: mlp.forward(x, plan=plan), lambda: mlp.forward(x[:3], adapters=ad, plan=plan),
           lambda: mlp.forward(x, adapters=pkg.MLPAdapters(w1=ad.w2), plan=plan),
           lambda: mlp.forward(x, adapters=pkg.MLPAdapters(w2=ad.w1), plan=plan),
           lambda: mlp.forward(x, adapters=ad, plan=pkg.lora_plan(torch.zeros(4, dtype=torch.int32, device=cuda), 2)),
           lambda: pkg.w4a8_mlp(pkg.quantize_mxint8(x), mlp.weights, adapters=ad, plan=plan),
           lambda: pkg.w4a8_mlp(x, mlp.weights, rows=x), lambda: pkg.w4a8_mlp(x, mlp.weights, residual=x[:2]),
           lambda: mlp.forward_add_rmsnorm(x, x[:2], w), lambda: mlp.forward_add_rmsnorm(x.half(), x, w),
           lambda: mlp.forward_add_rmsnorm(x, x, w[:64]), lambda: mlp.forward_add_rmsnorm(x[:, :64], x[:, :64], w),
           lambda: mlp.forward_add_rmsnorm(x, x, w, out=torch.empty(H, 4, dtype=torch.bfloat16, device=cuda).T),
           lambda: pkg.w4a8_mlp(x, pkg.Qwen36MLP(cuda, sd, weight_format="bf16", max_tokens=4).weights)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_argument_refusals_on_the_gpu(pkg, cuda):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda)
    wt = pkg.pack_weight(torch.ones(64, 64, dtype=torch.bfloat16, device=cuda), "mxfp4")
    n = torch.zeros(64, dtype=torch.bfloat16, device=cuda)
    t = pkg.quantize_mxint8(x)
    a, b = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda), torch.zeros(8, 4, dtype=torch.bfloat16, device=cuda)
    st, pl = pkg.pack_lora([(a, b, 1.0)]), pkg.lora_plan(torch.zeros(4, dtype=torch.int32, device=cuda), 1)
    f = torch.zeros(4, 64, device=cuda)
    o8 = torch.zeros(4, 8, device=cuda)
    calls = [
        lambda: pkg.w4a8_linear(t, wt, residual=x[:2]), lambda: pkg.w4a8_linear(t, wt, residual=x.half()),
        lambda: pkg.w4a8_linear(t, wt, out=f.half()), lambda: pkg.w4a8_linear(t, wt, out=f, out_dtype=torch.bfloat16),
        lambda: pkg.w4a8_linear(t, wt, out=f[:, :32]), lambda: pkg.w4a8_linear(t, wt, out=f, residual=x.view(-1)[:256].view(4, 64)[:3]),
        lambda: pkg.w4a8_linear(pkg.Mx8Tensor(t.buf[:100], 4, 64), wt), lambda: pkg.w4a8_linear(pkg.Mx8Tensor(t.buf, 4, 96), wt),
        lambda: pkg.w4a8_linear(t, pkg.pack_weight(torch.ones(64, 256, dtype=torch.bfloat16, device=cuda), "bfp8")),
        lambda: pkg.w4a8_linear(pkg.quantize_mxfp4(x), wt), lambda: pkg.w4a8_swiglu(t, wt, wt, quantize=True),
        lambda: pkg.w4a8_swiglu(t, wt, wt, gate_add=x), lambda: pkg.w4a8_swiglu(t, wt, wt, up_add=f[:2]),
        lambda: pkg.w4a8_swiglu(t, wt, wt, gate_add=f.T.contiguous()), lambda: pkg.w4a8_swiglu(t, wt, wt, gate_add=f.cpu()),
        lambda: pkg.add_rmsnorm(x, x[:2], n), lambda: pkg.add_rmsnorm(x, x.half(), n), lambda: pkg.add_rmsnorm(x.half(), x, n),
        lambda: pkg.add_rmsnorm(x, x, n.float()), lambda: pkg.add_rmsnorm(x, x, n[:32]), lambda: pkg.add_rmsnorm(x, None, n, out=x),
        lambda: pkg.add_rmsnorm(x, x, n, out=f), lambda: pkg.add_rmsnorm(x, x.clone(), n, out=x),
        lambda: pkg.add_rmsnorm(x, x.cpu(), n), lambda: pkg.add_rmsnorm(x, x.clone(), n, eps=-1.0), lambda: pkg.add_rmsnorm(x.T, x.T, n),
        lambda: pkg.lora_linear(x.half(), st, pl), lambda: pkg.lora_linear(x.float(), st, pl), lambda: pkg.lora_linear(x[:2], st, pl),
        lambda: pkg.lora_linear(x[:, :32], st, pl), lambda: pkg.lora_linear(x, st, pl, base=f), lambda: pkg.lora_linear(x, st, pl, base=o8.half()),
        lambda: pkg.lora_linear(x, st, pl, out=o8, out_dtype=torch.bfloat16), lambda: pkg.lora_linear(x, pl, st),
        lambda: pkg.lora_linear(x, st, pkg.lora_plan(torch.zeros(4, dtype=torch.int32, device=cuda), 2)),
        lambda: pkg.lora_plan(torch.zeros(4, dtype=torch.int64, device=cuda), 1), lambda: pkg.lora_plan(torch.zeros(2, 2, dtype=torch.int32, device=cuda), 1),
        lambda: pkg.lora_plan(torch.zeros(0, dtype=torch.int32, device=cuda), 1), lambda: pkg.lora_plan(torch.zeros(4, dtype=torch.int32, device=cuda), 0),
        lambda: pkg.pack_lora([(a, b, float("inf"))]), lambda: pkg.pack_lora([(a, b[:, :3].contiguous(), 1.0)]), lambda: pkg.pack_lora([(a, b, 1.0), (a.half(), b.half(), 1.0)]),
        lambda: pkg.pack_lora([(a.float(), b.float(), 1.0)]), lambda: pkg.pack_lora([(a[:, :48].contiguous(), b, 1.0)]),
        lambda: pkg.pack_lora([(torch.zeros(129, 64, dtype=torch.bfloat16, device=cuda), torch.zeros(8, 129, dtype=torch.bfloat16, device=cuda), 1.0)]),
        lambda: pkg.pack_lora([(a, b, 1.0), (a[:, :32].contiguous(), b, 1.0)]), lambda: pkg.pack_lora([(a.T, b, 1.0)]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)


def _run_all(pkg, mlp, ad, plan, x, r, w):
    h, rows, n = pkg.add_rmsnorm(x, r, w, output="both")
    y = pkg.w4a8_mlp(n, mlp.weights, residual=h, out_dtype=torch.float32, adapters=ad, plan=plan, rows=rows)
    return h, rows, pkg.dequantize(n), y


@pytest.mark.parametrize("M", [2, 40, 150])
def test_graphs_replay_what_eager_calls_compute(pkg, cuda, M):
    """Two graphs of a half layer with new inputs and new ids on every replay, eager work in between."""
    sd = _state(cuda, 3)
    mlp = pkg.Qwen36MLP(cuda, sd, weight_format="mxfp4", activation_format="mxint8", max_tokens=M)
    _, ad = _adapters(pkg, cuda, 1)
    g = torch.Generator().manual_seed(M)
    x, r = (torch.zeros(M, H, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    w = (torch.randn(H, generator=g) * 0.1).bfloat16().to(cuda)
    ids = torch.zeros(M, dtype=torch.int32, device=cuda)
    _run_all(pkg, mlp, ad, pkg.lora_plan(ids, 3), x, r, w)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            plan = pkg.lora_plan(ids, 3)
            outs = _run_all(pkg, mlp, ad, plan, x, r, w)
        graphs.append((gr, outs, plan))
    for _ in range(4):
        x.copy_(torch.randn(M, H, generator=g).bfloat16())
        r.copy_(torch.randn(M, H, generator=g).bfloat16())
        ids.copy_(torch.randint(-1, 4, (M,), generator=g, dtype=torch.int32))
        want = _run_all(pkg, mlp, ad, pkg.lora_plan(ids, 3), x, r, w)
        for gr, outs, _ in graphs:
            for o in outs:
                o.zero_()
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
        torch.empty(1 << 22, device=cuda).fill_(float("nan"))  # what the allocator hands out next is not zeros


def test_two_streams_share_a_plan_and_the_weights(pkg, cuda):
    sd = _state(cuda, 3)
    mlp = pkg.Qwen36MLP(cuda, sd, weight_format="mxfp4", activation_format="mxint8", max_tokens=64)
    _, ad = _adapters(pkg, cuda, 1)
    g = torch.Generator().manual_seed(2)
    for M in (20, 140):
        ids = torch.randint(-1, 4, (M,), generator=g, dtype=torch.int32).to(cuda)
        w = (torch.randn(H, generator=g) * 0.1).bfloat16().to(cuda)
        cases = [[torch.randn(M, H, generator=g).bfloat16().to(cuda) for _ in range(2)] for _ in range(2)]
        plan = pkg.lora_plan(ids, 3)
        want = [_run_all(pkg, mlp, ad, plan, x, r, w) for x, r in cases]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(5):
            for i, (s, (x, r)) in enumerate(zip(streams, cases)):
                with torch.cuda.stream(s):
                    got[i].append(_run_all(pkg, mlp, ad, plan, x, r, w))
        torch.cuda.synchronize()
        for i in range(2):
            for outs in got[i]:
                for a, b in zip(outs, want[i]):
                    assert torch.equal(a, b)


def test_every_call_on_a_given_stream(pkg, cuda):
    """``stream`` may be another one than the current one; what it returns is ready on that stream."""
    s = torch.cuda.Stream()
    g = torch.Generator().manual_seed(9)
    x, r = (torch.randn(70, 320, generator=g).bfloat16().to(cuda) for _ in range(2))
    w = torch.zeros(320, dtype=torch.bfloat16, device=cuda)
    pw = pkg.pack_weight((torch.randn(256, 320, generator=g) * 0.1).bfloat16().to(cuda), "mxfp4")
    raw = [(torch.randn(8, 320, generator=g).bfloat16().to(cuda), torch.randn(256, 8, generator=g).bfloat16().to(cuda), 1.0)]
    ids = torch.zeros(70, dtype=torch.int32, device=cuda)
    stack, plan, t = pkg.pack_lora(raw), pkg.lora_plan(ids, 1), pkg.quantize_mxint8(x)
    calls = [lambda **k: pkg.quantize_mxint8(x, **k).buf, lambda **k: pkg.add_rmsnorm(x, r, w, output="rows", **k)[1],
             lambda **k: pkg.add_rmsnorm(x, r, w, **k)[0], lambda **k: pkg.w4a8_linear(x, pw, **k),
             lambda **k: pkg.w4a8_swiglu(x, pw, pw, **k), lambda **k: pkg.dequantize(t, **k),
             lambda **k: pkg.unpack_canonical(t, **k)[0], lambda **k: pkg.lora_linear(x, stack, plan, **k),
             lambda **k: pkg.lora_linear(x, stack, pkg.lora_plan(ids, 1, **k), **k),
             lambda **k: pkg.pack_lora(raw, **k).b]
    for i, f in enumerate(calls):
        want = f()
        torch.cuda.synchronize()
        got = f(stream=s)
        s.synchronize()
        if i in (0,):  # bytes behind the last row are not written
            got, want = (pkg.dequantize(pkg.Mx8Tensor(b, 70, 320)) for b in (got, want))
        assert torch.equal(got, want), i
    assert torch.cuda.current_stream() != s


def test_rows_behind_the_last_one_stay(pkg, cuda):
    """Outputs in front of a guard: nothing behind the last row is written."""
    g = torch.Generator().manual_seed(3)
    for M, N in ((1, 33), (16, 100), (17, 65), (70, 257), (130, 320)):
        x = torch.randn(M, 96, generator=g).bfloat16().to(cuda)
        pw = pkg.pack_weight((torch.randn(N, 96, generator=g) * 0.1).bfloat16().to(cuda), "mxfp4")
        stack = pkg.pack_lora([(torch.randn(8, 96, generator=g).bfloat16().to(cuda), torch.randn(N, 8, generator=g).bfloat16().to(cuda), 1.0)])
        plan = pkg.lora_plan(torch.zeros(M, dtype=torch.int32, device=cuda), 1)
        for dt in (torch.bfloat16, torch.float32):
            for f in (lambda o: pkg.w4a8_linear(x, pw, out=o), lambda o: pkg.w4a8_swiglu(x, pw, pw, out=o),
                      lambda o: pkg.lora_linear(x, stack, plan, out=o)):
                flat = torch.full((M * N + 4096,), 3.0, dtype=dt, device=cuda)
                f(flat[:M * N].view(M, N))
                assert (flat[M * N:] == 3.0).all() and not (flat[:M * N] == 3.0).all()
        wide = torch.full((M + 8, 96 + 32), 3.0, dtype=torch.bfloat16, device=cuda)
        pkg.add_rmsnorm(x, x.clone(), torch.zeros(96, dtype=torch.bfloat16, device=cuda), out=wide[:M, :96])
        assert (wide[M:] == 3.0).all() and (wide[:, 96:] == 3.0).all()


@pytest.mark.parametrize("M", [1, 30, 130])
def test_tokens_without_an_adapter_beside_down_adapters(pkg, cuda, M):
    """With adapters of the down projection in a call every token's h is rounded to bf16 before it is quantised.  A token
    without one gets what the calls by themselves make of those rows, and 8-bit values at most one step (of the coarser
    of both scales) from those quantised from fp32: bf16 moves a value by at most a quarter of a step, rounding by half."""
    mlp = pkg.Qwen36MLP(cuda, _state(cuda, 7), weight_format="mxfp4", activation_format="mxint8", max_tokens=M)
    _, ad = _adapters(pkg, cuda, 2, which=("w2",))
    g = torch.Generator().manual_seed(M)
    x, res = torch.randn(M, H, generator=g).bfloat16().to(cuda), torch.randn(M, H, generator=g).to(cuda)
    plan = pkg.lora_plan(torch.full((M,), -1, dtype=torch.int32, device=cuda), 3)
    got = mlp.forward(x, residual=res, out_dtype=torch.float32, adapters=ad, plan=plan)
    rows = pkg.w4a8_swiglu(x, mlp.weights.w1, mlp.weights.w3)
    assert torch.equal(got, pkg.w4a8_linear(rows, mlp.weights.w2, residual=res, out_dtype=torch.float32))
    once, twice = pkg.w4a8_swiglu(x, mlp.weights.w1, mlp.weights.w3, quantize=True), pkg.quantize_mxint8(rows)
    scale = torch.maximum(*(pkg.unpack_canonical(t)[1] for t in (once, twice))).double()
    step = torch.exp2(scale - 133).repeat_interleave(32, dim=1)
    assert ((pkg.dequantize(once).double() - pkg.dequantize(twice).double()).abs() <= step).all()
