"""The differentiable functions without rows, and a Linear with adapters in a captured graph, on another stream, hooked and called by itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_no_rows():
    from comfyui_amd import autograd as A
    x = torch.empty((0, 64), device="cuda", dtype=BF16, requires_grad=True)
    w, b = (torch.ones(64, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2))
    A.layer_norm(x, w, b).sum().backward()
    assert x.grad.shape == (0, 64) and not w.grad.any() and not b.grad.any()
    a, ab = torch.ones((2, 8, 64), device="cuda", dtype=BF16, requires_grad=True), torch.ones((2, 32, 8), device="cuda", dtype=BF16, requires_grad=True)
    y = A.add_adapters(torch.empty((0, 32), device="cuda", dtype=BF16), x, a, ab, torch.ones(2, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"))
    y.sum().backward()
    assert y.shape == (0, 32) and not a.grad.any() and not ab.grad.any()


def linear(g):
    from comfyui_amd import ops
    lin = ops.disable_weight_init.Linear(640, 768, bias=False, dtype=BF16, device="cuda")
    with torch.no_grad():
        lin.weight.copy_(torch.randn(lin.weight.shape, generator=g, device="cuda") * 0.04)
    lin.adapters = ops.Adapters((torch.randn((3, 16, 640), generator=g, device="cuda") * 0.04).to(BF16), (torch.randn((3, 768, 16), generator=g, device="cuda") * 0.3).to(BF16),
                                torch.rand(3, generator=g, device="cuda") + 0.5)
    return lin


@pytest.mark.parametrize("requests,per", [(8, 1), (3, 300)])
@pytest.mark.parametrize("invariant", [False, True])
def test_a_linear_with_adapters_captured(requests, per, invariant):
    """Replays on rows and indices written anew, with eager calls between; the same on another stream."""
    g = torch.Generator(device="cuda").manual_seed(requests)
    lin = linear(g)
    lin.batch_invariant = invariant
    x = torch.randn((requests * per, 640), generator=g, device="cuda").to(BF16)
    lin.adapters.index = torch.zeros(requests, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        eager = lin(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            elsewhere = lin(x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(elsewhere, eager) and torch.equal(lin.forward(x), eager)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(x)
        for turn in range(3):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            lin.adapters.index.copy_(torch.randint(-1, 3, (requests,), generator=torch.Generator().manual_seed(turn)).to(torch.int32))
            graph.replay()
            want = lin(x)
            assert torch.equal(out, want), turn
            torch.cuda.synchronize()


def test_a_hooked_linear_with_adapters():
    """A pre-hook's input is the adapters' as well, and a hook's result the whole one."""
    from comfyui_amd import functional as HF
    g = torch.Generator(device="cuda").manual_seed(7)
    lin = linear(g)
    x = torch.randn((4, 10, 640), generator=g, device="cuda").to(BF16)
    index = torch.tensor([2, -1, 0, 1], dtype=torch.int32, device="cuda")
    lin.adapters.index, ad = index, lin.adapters
    with torch.no_grad():
        base = type(lin).forward(lin, 2 * x)
        want = HF.add_adapters(base, 2 * x, ad.a, ad.b, ad.scale, index)
        lin.register_forward_pre_hook(lambda m, args: (2 * args[0],))
        seen = []
        lin.register_forward_hook(lambda m, args, out: seen.append(out))
        assert torch.equal(lin(x), want) and seen[0] is not None and torch.equal(seen[0], want)
        ad.index = index[:1]
        assert torch.equal(lin(x[0, 0]), lin(x[0, :1])[0]) and lin(x[0, 0]).shape == (768,)
