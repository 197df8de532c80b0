"""Low-rank adapters at sizes that take every kernel of lora_linear (a test without a GPU holds the list to that),
against the formula in 64 bits, and the same outputs however many adapters are loaded.

The bound is that of tests/test_gpu_lora.py.  It holds for every path: a value's sum over K is rounded at most twice for
each 32 of it, four times where up to 16 waves' sums are added in pairs and seven times over up to 8 pieces, which is
less than the 50 roundings that it allows beyond K's."""
import pytest
import torch

from test_gpu_lora import _adapters, _check
from test_lora import FOUR, PATHS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(PATHS)))
def test_every_path(pkg, cuda, case, dtype):
    ids, ranks, N, K = PATHS[case]
    print(f"case lora {len(ids)} tokens, {len(ranks)} adapters up to {max(ranks)}, {N}x{K} {dtype}", flush=True)
    _check(pkg, cuda, ids, ranks, N, K, dtype, seed=100 + case)


@pytest.mark.parametrize("loaded", [4, 60, 120, 300, 1024])
def test_loaded_adapters_that_no_token_uses(pkg, cuda, loaded):
    """Four requests among adapters of which any number is loaded: A x in 8, 4, 2 and 1 pieces of K.  The sums are rounded
    in another order then, so they are compared with the formula, not with each other."""
    ids = [loaded - 1 - i for i in FOUR]
    _check(pkg, cuda, ids, [16] * loaded, 40, 4096, torch.bfloat16, seed=7)


def test_two_launches_on_a_given_stream_and_in_graphs(pkg, cuda):
    """The kernels of large ranks and few tokens, and of many loaded adapters, captured and replayed on new inputs and
    new ids, eager work in between."""
    g = torch.Generator().manual_seed(11)
    for M, L, r, N, K in ((3, 2, 128, 136, 5120), (520, 120, 16, 41, 4096)):
        stack = pkg.pack_lora([(a.to(cuda), b.to(cuda), s) for a, b, s in _adapters([r] * L, N, K, torch.bfloat16, 5)])
        x = torch.zeros(M, K, dtype=torch.bfloat16, device=cuda)
        ids = torch.zeros(M, dtype=torch.int32, device=cuda)
        pkg.lora_linear(x, stack, pkg.lora_plan(ids, L))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pkg.lora_linear(x, stack, pkg.lora_plan(ids, L))
        other = torch.cuda.Stream()
        for _ in range(4):
            x.copy_(torch.randn(M, K, generator=g).bfloat16())
            ids.copy_(torch.randint(-1, L + 1, (M,), generator=g, dtype=torch.int32))
            want = pkg.lora_linear(x, stack, pkg.lora_plan(ids, L))
            torch.cuda.synchronize()
            given = pkg.lora_linear(x, stack, pkg.lora_plan(ids, L, stream=other), stream=other)
            other.synchronize()
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(given, want)
            torch.empty(1 << 22, device=cuda).fill_(float("nan"))
