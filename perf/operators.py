"""The microscaled 4-bit (MXFP4) operators of this library, as cases that can be timed and compared.

A decoder whose checkpoint holds MXFP4 weights (32 consecutive K values share a power-of-two scale,
each value one of 0, .5, 1, 1.5, 2, 3, 4, 6 with a sign) quantises its activations the same way and
multiplies the two: ``quantize`` (an activation matrix to the format, and the values that it stands
for), ``linear`` (a projection with its residual add), ``swiglu`` (the gate/up pair with SiLU) and
``mlp`` (the whole feed-forward block, with the decoder's norm in front of it or a residual).

Fields of a case: ``kind``; ``tokens`` M; ``k`` (input features); ``n`` (output features; 0 for
"quantize"; the intermediate size for "mlp"); ``dtype`` of the activations ("bf16", "f16", "f32");
``residual``; ``norm`` ("mlp": ``forward_rmsnorm``); ``f32`` (an fp32 output instead of bf16).
"""
import math

import torch

own = False

H27, I27 = 5120, 17408  # the 27B layer
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
VALUE_BYTES = 17 / 32  # half a byte and a 32nd of a scale byte


def _case(kind, tokens, k, n=0, dtype="bf16", residual=False, norm=False, f32=False, name=None):
    c = {"kind": kind, "tokens": tokens, "k": k, "n": n, "dtype": dtype, "residual": residual, "norm": norm, "f32": f32}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one token's hidden state: launches and host time count
        _case("quantize", 1, H27, name="quantize-token"),
        # an odd number of rows of an fp32 residual stream
        _case("quantize", 777, H27, dtype="f32", name="quantize-rows777-f32"),
        # the intermediate activations of a full prefill chunk
        _case("quantize", 2048, I27, name="quantize-prefill"),
        # decode: the down projection of one token with its residual
        _case("linear", 1, I27, H27, residual=True, name="linear-decode1"),
        # a projection of a 16-token speculative verify block
        _case("linear", 16, H27, I27, name="linear-verify16"),
        # a short prompt of an odd length, the fp32 partial that an all-reduce takes
        _case("linear", 201, I27 // 2, H27, f32=True, name="linear-prompt201-f32"),
        # the down projection of a full prefill chunk
        _case("linear", 2048, I27, H27, residual=True, name="linear-prefill"),
        # decode: the gate/up pair of one token
        _case("swiglu", 1, H27, I27, name="swiglu-decode1"),
        # the gate/up pair of a 64-token verify window
        _case("swiglu", 64, H27, I27, name="swiglu-window64"),
        # the ragged last chunk of a longer prompt
        _case("swiglu", 777, H27, I27, dtype="f16", name="swiglu-prompt777"),
        # the feed-forward half of a decoder layer on a verify block, norm included
        _case("mlp", 16, H27, I27, norm=True, name="mlp-verify16"),
        # the block on a full prefill chunk
        _case("mlp", 2048, H27, I27, residual=True, name="mlp-prefill"),
    ]


def draw(rng):
    """Tokens spread over their logarithm from 1 to 2000; features: the 27B layer's, its two-way
    share's, or any multiples of the block (32; of 256 for the whole block) below them, for the
    products' output side any number."""
    kind = rng.choice(["quantize", "linear", "linear", "swiglu", "swiglu", "mlp"])
    tokens = int(math.exp(rng.uniform(0.0, math.log(2000))))

    def spread(step, most):
        return step * max(1, int(math.exp(rng.uniform(math.log(256 / step), math.log(most / step)))))

    if kind == "quantize":
        return _case(kind, tokens, rng.choice([H27, I27, I27 // 2, spread(32, I27)]), dtype=rng.choice(list(DTYPES)))
    if kind == "mlp":
        k, n = (H27, rng.choice([I27, I27 // 2])) if rng.random() < 0.4 else (spread(256, H27), spread(256, I27))
        norm = rng.random() < 0.5
        return _case(kind, tokens, k, n, residual=not norm and rng.random() < 0.7, norm=norm)
    if rng.random() < 0.4:
        k, n = rng.choice([(H27, I27), (H27, I27 // 2)])
        if kind == "linear" and rng.random() < 0.5:
            k, n = n, k
    else:
        k, n = spread(32, H27), spread(1, I27)
        if kind == "linear" and rng.random() < 0.5:
            k, n = spread(32, I27), spread(1, H27)
    return _case(kind, tokens, k, n, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                 residual=kind == "linear" and rng.random() < 0.5, f32=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs


def _tensors(case, seed):
    """Activations ~ N(0, 1) with an RMSNorm-like channel gain and a few channels eight times as
    large, weights ~ N(0, 0.02) (bf16 checkpoint values), norm weights around zero (the gain is 1 + w)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(7919 * seed + 29)
    M, K, N = case["tokens"], case["k"], case["n"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    gain = 0.5 + torch.rand((K,), generator=g, device="cuda", dtype=torch.float32)
    gain = torch.where(torch.rand((K,), generator=g, device="cuda") < 0.01, 8 * gain, gain)
    t = {"x": (normal(M, K) * gain).to(DTYPES[case["dtype"]])}
    out = K if case["kind"] == "mlp" else N
    if case["residual"]:
        t["residual"] = normal(M, out).bfloat16()
    if case["norm"]:
        t["norm"] = (normal(K) * 0.1).bfloat16()
    if case["kind"] == "linear":
        t["w"] = [(normal(N, K) * 0.02).bfloat16()]
    elif case["kind"] != "quantize":
        t["w"] = [(normal(N, K) * 0.02).bfloat16() for _ in range(2)]
    if case["kind"] == "mlp":
        t["w"].append((normal(K, N) * 0.02).bfloat16())
    return t


def _blocks(x):
    """Scaled 32-value blocks [rows, K / 32, 32] and their exponents: the block maximum's binade less 2."""
    v = x.float().reshape(x.shape[0], -1, 32)
    e = (torch.frexp(v.abs().amax(dim=2, keepdim=True))[1] - 1).clamp(min=-124) - 2
    return torch.ldexp(v, -e), e


def _code(v):
    """The index of the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even index, and the sign bit 8."""
    a = v.abs()
    up = [a > 0.25, a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5.0]
    return sum(u.to(torch.uint8) for u in up) + 8 * torch.signbit(v).to(torch.uint8)


def _quantize(x):
    """Codes (two to a byte, the first in the low half) [rows, K / 2] and scale bytes [rows, K / 32]."""
    v, e = _blocks(x)
    c = _code(v).reshape(x.shape)
    return c[:, 0::2] | (c[:, 1::2] << 4), (e.squeeze(2) + 127).to(torch.uint8)


def _values(codes, scales):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    c = torch.stack([codes & 15, codes >> 4], dim=2).reshape(codes.shape[0], -1, 32)
    return torch.ldexp(table[c.int()], scales.int().unsqueeze(2) - 127).reshape(codes.shape[0], -1)


def prepare(case, seed):
    t = _tensors(case, seed)
    state = {"case": case, "x": t["x"], "residual": t.get("residual"), "norm": t.get("norm")}
    if case["kind"] == "quantize":
        return state
    # the checkpoint's MXFP4 matrices: codes and scales; a program that calls the library packs them at load
    canonical = [_quantize(w) for w in t["w"]]
    if own:
        import __graft_entry__

        pkg = __graft_entry__.load_package()
        if case["kind"] == "mlp":
            names = ("gate_proj", "up_proj", "down_proj")
            state["mlp"] = pkg.Qwen36MLP("cuda", {f"{n}.weight": w for n, w in zip(names, t["w"])},
                                         weight_format="mxfp4", max_tokens=case["tokens"])
        else:
            state["w"] = [pkg.pack_canonical(c, s, "mxfp4") for c, s in canonical]
    else:
        state["w"] = canonical
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    kind, dtype = case["kind"], torch.float32 if case["f32"] else torch.bfloat16
    x = state["x"]
    if own:
        import __graft_entry__

        pkg = __graft_entry__.load_package()
        if kind == "quantize":
            return pkg.dequantize(pkg.quantize_mxfp4(x), dtype=torch.bfloat16)
        if kind == "linear":
            return pkg.mxfp4_linear(x, state["w"][0], residual=state["residual"], out_dtype=dtype)
        if kind == "swiglu":
            return pkg.mxfp4_swiglu(x, *state["w"], out_dtype=dtype)
        if case["norm"]:
            return state["mlp"].forward_rmsnorm(x, state["norm"], eps=EPS, out_dtype=dtype)
        return state["mlp"].forward(x, residual=state["residual"], out_dtype=dtype)
    residual = state["residual"]
    if case["norm"]:
        residual, f = x, x.float()
        f = f * torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS) * (1 + state["norm"].float())
        x = f.bfloat16()
    v = _values(*_quantize(x))
    if kind == "quantize":
        return v.to(torch.bfloat16)
    w = [_values(*q) for q in state["w"]]
    y = v @ w[0].T
    if kind != "linear":
        y = y / (1 + torch.exp(-y)) * (v @ w[1].T)
    if kind == "mlp":
        y = _values(*_quantize(y)) @ w[2].T
    if residual is not None:
        y = y + residual.float()
    return y.to(dtype)


def work(case):
    M, K, N = case["tokens"], case["k"], case["n"]
    x = M * K * DTYPES[case["dtype"]].itemsize
    size = 4 if case["f32"] else 2
    if case["kind"] == "quantize":
        return {"bytes": x + 2 * M * K, "flops": 2 * M * K}
    matrices = {"linear": 1, "swiglu": 2, "mlp": 3}[case["kind"]]
    out = K if case["kind"] == "mlp" else N
    rows = x + M * out * (size + (2 if case["residual"] else 0)) + (2 * K if case["norm"] else 0)
    return {"bytes": matrices * N * K * VALUE_BYTES + rows, "flops": 2 * matrices * M * N * K}


# ---------------------------------------------------------------- the definition in 64 bits


def _exact_values(x):
    """What the format makes of x, from its definition: the block's scale is the power of two that puts
    its largest value into [4, 8); a value is rounded half to even to the element's two significant
    bits, to halves below 1, and to 6 where it would pass it."""
    v = x.double().reshape(x.shape[0], -1, 32)
    top = v.abs().amax(dim=2, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -124))) - 2)
    a = (v / scale).abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=1.0))) - 1)
    r = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.sign(v) * r * scale).reshape(x.shape)


def exact(case, seed):
    t = _tensors(case, seed)
    x, residual = t["x"], t.get("residual")
    if case["norm"]:
        residual, d = x, x.double()
        d = d / torch.sqrt((d * d).sum(dim=1, keepdim=True) / case["k"] + EPS) * (1 + t["norm"].double())
        x = d.bfloat16()  # the norm hands the block a bf16 tensor
    v = _exact_values(x)
    if case["kind"] == "quantize":
        return v
    w = [_exact_values(m) for m in t["w"]]
    y = torch.mm(v, w[0].T)
    if case["kind"] != "linear":
        y = y * torch.sigmoid(y) * torch.mm(v, w[1].T)
    if case["kind"] == "mlp":
        y = torch.mm(_exact_values(y), w[2].T)
    return y if residual is None else y + residual.double()
