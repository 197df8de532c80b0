"""The operators around a block of 4-bit weights and 8-bit activations, as cases that can be timed and
compared.

A server that keeps its projections in MXFP4 (32 consecutive K values share a power-of-two scale) and
wants more of the activations than 4 bits runs, for each half of a decoder layer: ``norm`` (the
attention's output added to the residual stream, the zero-centred RMSNorm of the sum, and that in
MXINT8: 8-bit integers, 32 to a power-of-two scale), ``linear`` and ``swiglu`` (products of 8-bit
activations and 4-bit weights), and beside each projection ``lora`` (the low-rank adapters of many
requests at once).

Fields of a case: ``kind``; ``tokens`` M; ``k`` (input features); ``n`` (output features; 0 for "norm");
``dtype`` of the activations ("bf16", "f16", "f32"); ``residual`` ("bf16", "f32" or "": what is added:
the residual stream of "norm", the residual of "linear", the base of "lora"); ``f32`` (an fp32 output
instead of bf16).  "lora" too: ``requests`` that the tokens belong to, in runs of equal length;
``adapters`` that are loaded; ``rank`` of the largest of them; ``ragged`` (every second adapter has a
smaller rank).
"""
import math

import torch

own = False

H27, I27 = 5120, 17408  # the 27B layer
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
VALUE_BYTES = 17 / 32  # of a 4-bit weight: half a byte and a 32nd of a scale byte


def _case(kind, tokens, k, n=0, dtype="bf16", residual="", f32=False, requests=0, adapters=0, rank=0, ragged=False,
          name=None):
    c = {"kind": kind, "tokens": tokens, "k": k, "n": n, "dtype": dtype, "residual": residual, "f32": f32,
         "requests": requests, "adapters": adapters, "rank": rank, "ragged": ragged}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one token between attention and feed-forward: launches and host time count
        _case("norm", 1, H27, residual="bf16", name="norm-token"),
        # an odd number of rows: an fp32 partial of the attention on an fp32 residual stream
        _case("norm", 777, H27, dtype="f32", residual="f32", name="norm-rows777-f32"),
        # a full prefill chunk
        _case("norm", 2048, H27, residual="bf16", name="norm-prefill"),
        # decode: the down projection of one token with its residual
        _case("linear", 1, I27, H27, residual="bf16", name="linear-decode1"),
        # a short prompt of an odd length, the fp32 partial that an all-reduce takes
        _case("linear", 201, I27 // 2, H27, f32=True, name="linear-prompt201-f32"),
        # the down projection of a full prefill chunk
        _case("linear", 2048, I27, H27, residual="bf16", name="linear-prefill"),
        # the gate/up pair of a 16-token speculative verify block
        _case("swiglu", 16, H27, I27, name="swiglu-verify16"),
        # the ragged last chunk of a longer prompt
        _case("swiglu", 777, H27, I27, dtype="f16", name="swiglu-prompt777"),
        # one token of one request beside the down projection's residual
        _case("lora", 1, I27, H27, residual="bf16", requests=1, adapters=4, rank=16, name="lora-decode1"),
        # 32 requests decode one token each, eleven adapters among them, beside the gate projection
        _case("lora", 32, H27, I27, requests=32, adapters=12, rank=32, ragged=True, f32=True, name="lora-batch32"),
        # five verify windows of odd length, an odd rank
        _case("lora", 85, H27, H27 + 1, dtype="f16", residual="f32", requests=5, adapters=3, rank=24, f32=True,
              name="lora-windows85"),
        # prompts of four requests in one prefill chunk, beside the down projection
        _case("lora", 2048, I27, H27, residual="bf16", requests=4, adapters=8, rank=64, name="lora-prefill"),
    ]


def draw(rng):
    """Tokens spread over their logarithm from 1 to 2000; features: the 27B layer's, its two-way share's,
    or any multiples of 32 below them, for the outputs any number; ranks from 1 to 128."""
    kind = rng.choice(["norm", "linear", "swiglu", "lora", "lora"])
    tokens = int(math.exp(rng.uniform(0.0, math.log(2000))))

    def spread(step, most):
        return step * max(1, int(math.exp(rng.uniform(math.log(256 / step), math.log(most / step)))))

    if kind == "norm":
        return _case(kind, tokens, rng.choice([H27, spread(32, H27), spread(32, I27)]),
                     dtype=rng.choice(["bf16", "bf16", "f32"]), residual=rng.choice(["bf16", "bf16", "f32"]))
    if rng.random() < 0.4:
        k, n = rng.choice([(H27, I27), (H27, I27 // 2)])
    else:
        k, n = spread(32, H27), spread(1, I27)
    if kind != "swiglu" and rng.random() < 0.5:
        k, n = (n, k) if n % 32 == 0 else (spread(32, I27), spread(1, H27))
    residual, f32 = rng.choice(["", "bf16", "f32"]), rng.random() < 0.3
    if kind == "lora":
        requests = min(tokens, int(math.exp(rng.uniform(0.0, math.log(64)))))
        return _case(kind, tokens, k, n, dtype=rng.choice(["bf16", "bf16", "f16"]), residual=residual, f32=f32,
                     requests=requests, adapters=rng.randint(1, 24), rank=int(math.exp(rng.uniform(0.0, math.log(128)))),
                     ragged=rng.random() < 0.5)
    return _case(kind, tokens, k, n, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                 residual=residual if kind == "linear" else "", f32=f32)


# ---------------------------------------------------------------- inputs


def _adapter_of(case):
    """The adapter of each request before a seed renames the adapters: one request in eight has none (-1)."""
    return [-1 if i % 8 == 5 else (5 * i + 1) % case["adapters"] for i in range(case["requests"])]


def _ranks(case):
    return [max(1, case["rank"] // 2 - a % 3) if case["ragged"] and a % 2 else case["rank"]
            for a in range(case["adapters"])]


def _request_of(case):
    """The request that each token belongs to."""
    M, R = case["tokens"], case["requests"]
    return [t * R // M for t in range(M)]


def _tensors(case, seed):
    """Activations ~ N(0, 1) with an RMSNorm-like channel gain and a few channels eight times as large,
    weights ~ N(0, 0.02), norm weights around zero (the gain is 1 + w); adapters as training leaves them, A
    ~ N(0, 1 / sqrt(K)), B ~ N(0, 0.02), scale alpha / rank."""
    g = torch.Generator(device="cuda")
    g.manual_seed(7919 * seed + 31)
    M, K, N, kind = case["tokens"], case["k"], case["n"], case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    gain = 0.5 + torch.rand((K,), generator=g, device="cuda", dtype=torch.float32)
    gain = torch.where(torch.rand((K,), generator=g, device="cuda") < 0.01, 8 * gain, gain)
    t = {"x": (normal(M, K) * gain).to(DTYPES[case["dtype"]])}
    if case["residual"]:
        t["residual"] = normal(M, K if kind == "norm" else N).to(DTYPES[case["residual"]])
    if kind == "norm":
        t["norm"] = (normal(K) * 0.1).bfloat16()
    elif kind == "lora":
        names = torch.randperm(case["adapters"], generator=torch.Generator().manual_seed(seed + 1)).tolist()
        t["ids"] = torch.tensor([names[a] if a >= 0 else -1
                                 for a in map(_adapter_of(case).__getitem__, _request_of(case))],
                                dtype=torch.int32, device="cuda")
        t["adapters"] = [None] * case["adapters"]
        for a, r in enumerate(_ranks(case)):
            t["adapters"][names[a]] = ((normal(r, K) / math.sqrt(K)).to(DTYPES[case["dtype"]]),
                                       (normal(N, r) * 0.02).to(DTYPES[case["dtype"]]), 2.0 * (1 + a % 4) / r)
    else:
        t["w"] = [(normal(N, K) * 0.02).bfloat16() for _ in range(2 if kind == "swiglu" else 1)]
    return t


def _weight_codes(w):
    """Codes (two to a byte, the first in the low half) [rows, K / 2] and scale bytes [rows, K / 32] of a
    checkpoint's MXFP4 matrix: the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even index."""
    v = w.float().reshape(w.shape[0], -1, 32)
    e = (torch.frexp(v.abs().amax(dim=2, keepdim=True))[1] - 1).clamp(min=-124) - 2
    v = torch.ldexp(v, -e)
    a = v.abs()
    up = [a > 0.25, a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5.0]
    c = sum(u.to(torch.uint8) for u in up) + 8 * torch.signbit(v).to(torch.uint8)
    c = c.reshape(w.shape)
    return c[:, 0::2] | (c[:, 1::2] << 4), (e.squeeze(2) + 127).to(torch.uint8)


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def prepare(case, seed):
    t = _tensors(case, seed)
    state = {"case": case, "x": t["x"], "residual": t.get("residual"), "norm": t.get("norm")}
    if case["kind"] == "lora":
        if own:
            # the adapters are packed when they are loaded; the plan says which tokens share one, and serves
            # every projection of every layer in this step
            state["lora"] = _package().pack_lora(t["adapters"])
            state["plan"] = _package().lora_plan(t["ids"], case["adapters"])
        else:
            state["ids"], most = t["ids"], max(_ranks(case))
            pad = [most - a.shape[0] for a, _, _ in t["adapters"]]
            state["a"] = torch.stack([torch.nn.functional.pad(a, (0, 0, 0, p)) for (a, _, _), p in zip(t["adapters"], pad)])
            state["b"] = torch.stack([torch.nn.functional.pad(b, (0, p)) for (_, b, _), p in zip(t["adapters"], pad)])
            state["scale"] = torch.tensor([s for _, _, s in t["adapters"]], device="cuda")
    elif case["kind"] != "norm":
        # the checkpoint's MXFP4 matrices; a program that calls the library packs them at load
        state["w"] = [_weight_codes(w) for w in t["w"]]
        if own:
            state["w"] = [_package().pack_canonical(c, s, "mxfp4") for c, s in state["w"]]
    return state


# ---------------------------------------------------------------- one pass


def _mxint8(x):
    """The values that MXINT8 makes of x: 127 steps to either side, the step a 64th of the binade of the
    block's maximum; rounded half to even, 128 steps to 127."""
    v = x.float().reshape(x.shape[0], -1, 32)
    e = (torch.frexp(v.abs().amax(dim=2, keepdim=True))[1] - 1).clamp(-120, 126) - 6
    return torch.ldexp(torch.round(torch.ldexp(v, -e)).clamp(-127.0, 127.0), e).reshape(x.shape)


def _weight_values(codes, scales):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    c = torch.stack([codes & 15, codes >> 4], dim=2).reshape(codes.shape[0], -1, 32)
    return torch.ldexp(table[c.int()], scales.int().unsqueeze(2) - 127).reshape(codes.shape[0], -1)


def run(state):
    case = state["case"]
    kind, dtype = case["kind"], torch.float32 if case["f32"] else torch.bfloat16
    x, residual = state["x"], state["residual"]
    if own:
        pkg = _package()
        if kind == "norm":
            h, n = pkg.add_rmsnorm(x, residual, state["norm"], eps=EPS, output="mxint8")
            return h, pkg.dequantize(n, dtype=torch.bfloat16)
        if kind == "linear":
            return pkg.w4a8_linear(x, state["w"][0], residual=residual, out_dtype=dtype)
        if kind == "swiglu":
            return pkg.w4a8_swiglu(x, *state["w"], out_dtype=dtype)
        return pkg.lora_linear(x, state["lora"], state["plan"], base=residual, out_dtype=dtype)
    if kind == "norm":
        h = (x.float() + residual.float()).to(residual.dtype)
        f = h.float()
        f = f * torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS) * (1 + state["norm"].float())
        return h, _mxint8(f.bfloat16()).bfloat16()
    if kind == "lora":
        L, R, K = state["a"].shape
        mine = (state["ids"].unsqueeze(1) == torch.arange(L, device=x.device)) * state["scale"]
        s = (x.float() @ state["a"].float().reshape(L * R, K).T).reshape(-1, L, R) * mine.unsqueeze(2)
        y = s.reshape(-1, L * R) @ state["b"].float().permute(0, 2, 1).reshape(L * R, -1)
    else:
        v = _mxint8(x)
        w = [_weight_values(*q) for q in state["w"]]
        y = v @ w[0].T
        if kind == "swiglu":
            y = y / (1 + torch.exp(-y)) * (v @ w[1].T)
    if residual is not None:
        y = y + residual.float()
    return y.to(dtype)


def work(case):
    M, K, N, kind = case["tokens"], case["k"], case["n"], case["kind"]
    x = M * K * DTYPES[case["dtype"]].itemsize
    added = DTYPES[case["residual"]].itemsize if case["residual"] else 0
    if kind == "norm":
        return {"bytes": x + M * K * (2 * added + 2) + 2 * K, "flops": 8 * M * K}
    rows = x + M * N * ((4 if case["f32"] else 2) + added)
    if kind == "lora":
        ranks, used = _ranks(case), _adapter_of(case)
        values = sum(ranks[a] for a in set(used) if a >= 0) * (K + N)
        flops = sum(2 * ranks[used[r]] * (K + N) for r in _request_of(case) if used[r] >= 0)
        return {"bytes": rows + values * DTYPES[case["dtype"]].itemsize, "flops": flops}
    matrices = 2 if kind == "swiglu" else 1
    return {"bytes": matrices * N * K * VALUE_BYTES + rows, "flops": 2 * matrices * M * N * K}


# ---------------------------------------------------------------- the definition in 64 bits


def _exact_mxfp4(w):
    v = w.double().reshape(w.shape[0], -1, 32)
    top = v.abs().amax(dim=2, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -124))) - 2)
    a = (v / scale).abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=1.0))) - 1)
    r = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.sign(v) * r * scale).reshape(w.shape)


def _exact_mxint8(x):
    v = x.double().reshape(x.shape[0], -1, 32)
    top = v.abs().amax(dim=2, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120)))) / 64
    return (torch.round(v / step).clamp(-127.0, 127.0) * step).reshape(x.shape)


def exact(case, seed):
    t = _tensors(case, seed)
    x, residual = t["x"], t.get("residual")
    if case["kind"] == "norm":
        h = (x.double() + residual.double()).to(residual.dtype)  # the residual stream keeps its type
        d = h.double()
        d = d / torch.sqrt((d * d).sum(dim=1, keepdim=True) / case["k"] + EPS) * (1 + t["norm"].double())
        return x.double() + residual.double(), _exact_mxint8(d.bfloat16())  # the norm hands over bf16 values
    if case["kind"] == "lora":
        y = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device="cuda")
        for a, (down, up, scale) in enumerate(t["adapters"]):
            rows = torch.nonzero(t["ids"] == a).squeeze(1)
            if len(rows):
                y[rows] = scale * torch.mm(torch.mm(x[rows].double(), down.double().T), up.double().T)
    else:
        v = _exact_mxint8(x)
        w = [_exact_mxfp4(m) for m in t["w"]]
        y = torch.mm(v, w[0].T)
        if case["kind"] == "swiglu":
            y = y * torch.sigmoid(y) * torch.mm(v, w[1].T)
    return y if residual is None else y + residual.double()
