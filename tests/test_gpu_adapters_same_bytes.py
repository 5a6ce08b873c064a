"""Adapters beside a Linear with batch_invariant: a row has the same bytes whatever rows come with it, as the Linear's own product has."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def linear(g, K, N, n, R, dtype, invariant=True):
    from comfyui_amd import ops
    lin = ops.disable_weight_init.Linear(K, N, bias=False, dtype=dtype, device="cuda")
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    with torch.no_grad():
        lin.weight.copy_(rand(N, K) * K ** -0.5)
    lin.adapters = ops.Adapters((rand(n, R, K) * K ** -0.5).to(dtype), (rand(n, N, R) * 0.3).to(dtype), torch.rand(n, generator=g, device="cuda") + 0.5)
    lin.batch_invariant = invariant
    return lin


def call(lin, x, index):
    lin.adapters.index = index.to(torch.int32).cuda()
    with torch.no_grad():
        return lin(x)


@pytest.mark.parametrize("dtype", [BF16, torch.float16])
@pytest.mark.parametrize("K,N,n,R", [(6912, 2560, 3, 16), (2560, 1280, 3, 40), (5120, 768, 2, 96), (2176, 512, 70, 8), (4096, 256, 2, 200)])
def test_a_row_among_others(dtype, K, N, n, R):
    """Alone, among 48 rows of as many requests, among 600 and 2500 rows of one request, of requests of 20 rows each, and of requests of one row."""
    g = torch.Generator(device="cuda").manual_seed(K + R)
    lin = linear(g, K, N, n, R, dtype)
    x = (torch.randn((2500, K), generator=g, device="cuda") * torch.exp(0.7 * torch.randn(K, generator=g, device="cuda"))).to(dtype)
    alone = call(lin, x[7:8], torch.tensor([1]))
    other = torch.randint(-1, n, (2500,), generator=torch.Generator().manual_seed(R))
    other[7] = 1
    got = {"16": call(lin, x[:16], torch.tensor([1])), "48": call(lin, x[:48], other[:48]), "600": call(lin, x[:600], torch.tensor([1])), "2500": call(lin, x, torch.tensor([1])),
           "600 of 20": call(lin, x[:600], torch.cat([torch.tensor([1]), other[1:30]])), "2500 each": call(lin, x, other), "100 each": call(lin, x[:100], other[:100])}
    for what, y in got.items():
        assert torch.equal(y[7], alone[0]), what
    assert torch.equal(got["600"], got["2500"][:600]) and torch.equal(got["100 each"], got["2500 each"][:100])


def test_routed_experts_among_others():
    """An expert's Linears that ask for it, called on their rows alone or among those of other tokens."""
    from comfyui_amd import hidream, ops
    g = torch.Generator(device="cuda").manual_seed(3)
    ff = hidream.FeedForwardSwiGLU(2560, 3200, dtype=BF16, device="cuda")
    with torch.no_grad():
        for l in (ff.w1, ff.w2, ff.w3):
            l.weight.copy_(torch.randn(l.weight.shape, generator=g, device="cuda") * 0.02)
            N, K = l.weight.shape
            l.adapters = ops.Adapters((torch.randn((2, 16, K), generator=g, device="cuda") * K ** -0.5).to(BF16),
                                      (torch.randn((2, N, 16), generator=g, device="cuda") * 0.3).to(BF16), torch.ones(2, device="cuda"))
            l.adapters.index = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
            l.batch_invariant = True
        x = torch.randn((600, 2560), generator=g, device="cuda").to(BF16)
        perm = torch.randperm(1200, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        rows = x[(perm // 2).long()]
        with ops.routed_adapters(ff, 600, perm):
            whole = ff(rows)
        for lo, hi in ((0, 1), (0, 40), (5, 333), (100, 1100)):
            with ops.routed_adapters(ff, 600, perm[lo:hi]):
                assert torch.equal(ff(rows[lo:hi].contiguous()), whole[lo:hi]), (lo, hi)


def test_the_functions_own_flag():
    """functional.add_adapters(fixed_k_cut=True) with and without the compiled call."""
    from comfyui_amd import functional as HF
    from tests.test_gpu_adapters import problem
    p = problem(3, 600, 1, 6912, 256, 3, 16, BF16)
    rest = [p[k] for k in ("x", "a", "b", "scale", "index")]
    whole = HF.add_adapters(p["base"], *rest, fixed_k_cut=True)
    for lo, hi in ((0, 1), (3, 50), (100, 400)):
        part = [p["x"][lo:hi], p["a"], p["b"], p["scale"], p["index"][lo:hi]]
        calls, made = HF._row_calls, []
        try:
            for c in (calls, None):
                HF._row_calls = c
                made.append(HF.add_adapters(p["base"][lo:hi], *part, fixed_k_cut=True))
        finally:
            HF._row_calls = calls
        assert torch.equal(made[0], whole[lo:hi]) and torch.equal(made[0], made[1])
