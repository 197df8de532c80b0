"""Loading a layer without a GPU: what ``load_mlp_weights`` does around its conversions, with the
conversion and its check replaced by stand-ins."""
import weakref

import pytest
import torch

I, H = 512, 256


class _Source(torch.Tensor):
    """A checkpoint tensor whose device copy is a tensor of this process, kept in ``copies`` weakly."""

    copies = []

    def to(self, *args, **kwargs):
        t = torch.zeros(tuple(self.shape), dtype=torch.bfloat16)
        _Source.copies.append(weakref.ref(t))
        return t


class _Checkpoint(dict):
    """Makes a tensor at each access and keeps none, like a lazily read checkpoint."""

    def __getitem__(self, name):
        return torch.zeros(super().__getitem__(name)).as_subclass(_Source)


def _checkpoint():
    return _Checkpoint({"gate_proj.weight": (I, H), "up_proj.weight": (I, H), "down_proj.weight": (H, I)})


@pytest.fixture
def stand_ins(pkg, monkeypatch):
    from qwen_mlp_amd import mlp

    def begin(w, fmt, stream):
        return mlp.PackedWeight(torch.zeros(0, dtype=torch.uint8), *w.shape, fmt)

    monkeypatch.setattr(_Source, "copies", [])
    monkeypatch.setattr(mlp, "_pack_weight_begin", begin)
    monkeypatch.setattr(mlp, "_pack_weight_end", lambda pw, strict, stream: pw)
    return mlp


def test_sources_outlive_their_conversions(stand_ins, monkeypatch):
    """A matrix's bf16 source lives until the check that waits for its conversion: dropped before,
    memory that belongs to another stream could be handed out again while the conversion reads it."""
    mlp = stand_ins
    alive = []

    def end(pw, strict, stream):
        alive.append(_Source.copies[len(alive)]() is not None)
        return pw

    monkeypatch.setattr(mlp, "_pack_weight_end", end)
    mlp.load_mlp_weights("cuda", _checkpoint())
    assert alive == [True, True, True]


def test_a_later_failure_keeps_what_came_before(stand_ins, monkeypatch, tmp_path):
    """Matrices load in the order gate, down, up: where a later one is missing, those before it
    have been checked and cached, and where one of those is refused, that is the error."""
    mlp = stand_ins
    from qwen_mlp_amd import weight_cache

    saved = []
    monkeypatch.setattr(weight_cache, "save", lambda path, pw: saved.append((pw.rows, pw.cols)))
    sd = _checkpoint()
    del sd["up_proj.weight"]
    with pytest.raises(KeyError, match="up_proj"):
        mlp.load_mlp_weights("cuda", sd, tensor_cache_path=str(tmp_path))
    assert saved == [(I, H), (H, I)]

    def end(pw, strict, stream):
        raise ValueError("non-finite")

    monkeypatch.setattr(mlp, "_pack_weight_end", end)
    with pytest.raises(ValueError, match="non-finite"):
        mlp.load_mlp_weights("cuda", sd, tensor_cache_path=str(tmp_path))


def test_pool_refuses_a_device_that_is_not_a_gpu(pkg, monkeypatch):
    """Also where the current GPU's stream already holds a workspace."""
    from qwen_mlp_amd import _lib

    pool = pkg.WorkspacePool()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_lib, "raw_stream", lambda index=None: 0)
    pool._ws[pool._key("cuda", None)] = torch.zeros(64, dtype=torch.uint8)
    assert pool.reserve(64, "cuda:0").numel() == 64
    with pytest.raises(ValueError, match="cpu"):
        pool.reserve(64, "cpu")


class _OnGpu1(torch.Tensor):
    """Host memory that says it is on the second GPU."""

    @property
    def device(self):
        return torch.device("cuda", 1)

    def get_device(self):
        return 1


class _Calls:
    """A library whose calls succeed; ``made`` holds (name, current GPU, stream) of each."""

    def __init__(self):
        self.made, self.current = [], 0

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_bytes"):
                return 64
            self.made.append((name, self.current, args[-1]))
            return 0

        return call


@pytest.fixture
def calls(pkg, monkeypatch):
    """The first GPU is current; GPU i's current stream has the handle 100 + i."""
    from qwen_mlp_amd import _lib

    c = _Calls()

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, c.current = c.current, self.index

        def __exit__(self, *exc):
            c.current = self.before

    empty = torch.empty
    monkeypatch.setattr(_lib, "lib", lambda: c)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: c.current)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: c.current)
    monkeypatch.setattr(torch, "empty", lambda *size, device=None, **kw: empty(*size, **kw).as_subclass(_OnGpu1))
    return c


@pytest.mark.parametrize("fmt", ["bf16", "bfp8", "bf4", "mxfp4"])
def test_a_weight_is_packed_and_checked_on_its_own_gpu(pkg, calls, fmt):
    from qwen_mlp_amd import mlp

    w = torch.zeros(16, 256, dtype=torch.bfloat16).as_subclass(_OnGpu1)
    pw = pkg.pack_weight(w, fmt)
    mlp._read_info(pw)
    assert [name for name, *_ in calls.made] == ["qmlp_quantize_pack", "qmlp_quantize_pack_info", "qmlp_packed_info"]
    assert [(gpu, getattr(stream, "value", stream)) for _, gpu, stream in calls.made] == 3 * [(1, 101)]
    assert calls.current == 0


@pytest.mark.parametrize("fmt", ["bf16", "bfp8", "bf4", "mxfp4"])
def test_the_block_runs_on_its_input_gpu(pkg, calls, fmt):
    def tensor(*size, dtype=torch.bfloat16):
        return torch.zeros(*size, dtype=dtype).as_subclass(_OnGpu1)

    gate_up, down = pkg.matrix_formats(fmt)
    buf = tensor(64, dtype=torch.uint8)
    w = pkg.MLPWeights(w1=pkg.PackedWeight(buf, I, H, gate_up), w3=pkg.PackedWeight(buf, I, H, gate_up),
                       w2=pkg.PackedWeight(buf, H, I, down))
    x, norm = tensor(4, H), tensor(H)
    for workspace in (None, buf):
        pkg.mlp_forward(x, w, residual=x, workspace=workspace)
        pkg.mlp_forward_rmsnorm(x, norm, w, workspace=workspace)
    assert [name for name, *_ in calls.made] == ["qmlp_workspace_init", "qmlp_forward_ex", "qmlp_workspace_init",
                                                 "qmlp_forward_rmsnorm", "qmlp_forward_ex", "qmlp_forward_rmsnorm"]
    assert [(gpu, getattr(stream, "value", stream)) for _, gpu, stream in calls.made] == 6 * [(1, 101)]
    assert calls.current == 0


class _OnGpu0(torch.Tensor):
    @property
    def device(self):
        return torch.device("cuda", 0)

    def get_device(self):
        return 0


def test_the_block_refuses_tensors_of_two_gpus(pkg, calls):
    """A kernel that is given another GPU's pointer may fault; nothing is launched."""
    def tensor(*size, dtype=torch.bfloat16, gpu=_OnGpu1):
        return torch.zeros(*size, dtype=dtype).as_subclass(gpu)

    def weights(other=None):
        bufs = {n: tensor(64, dtype=torch.uint8, gpu=_OnGpu0 if n == other else _OnGpu1) for n in ("w1", "w2", "w3")}
        return pkg.MLPWeights(**{n: pkg.PackedWeight(b, *((H, I) if n == "w2" else (I, H)), "mxfp4") for n, b in bufs.items()})

    x, norm, there = tensor(4, H), tensor(H), tensor(4, H, gpu=_OnGpu0)
    for name in ("w1", "w2", "w3"):
        for f in (lambda w: pkg.mlp_forward(x, w), lambda w: pkg.mlp_forward_rmsnorm(x, norm, w)):
            with pytest.raises(ValueError, match=f"{name} is on cuda:0, x on cuda:1"):
                f(weights(name))
    for kw in (dict(residual=there), dict(out=there), dict(workspace=there)):
        with pytest.raises(ValueError, match="is on cuda:0"):
            pkg.mlp_forward(x, weights(), **kw)
        if "residual" not in kw:
            with pytest.raises(ValueError, match="is on cuda:0"):
                pkg.mlp_forward_rmsnorm(x, norm, weights(), **kw)
    with pytest.raises(ValueError, match="norm_weight"):
        pkg.mlp_forward_rmsnorm(x, tensor(H, gpu=_OnGpu0), weights())
    assert calls.made == []
