"""The router's balance loss, counts and gradients against 64 bits (tests/router64.py derives the tolerances)."""
import pytest
import torch

from tests import router64
from tests.norm64 import close

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def problem(seed, S, L, D, E, k, dtype, masked=False, weights=True):
    g = gen(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    T = S * L
    x = (rand(T, D) * torch.exp(0.7 * rand(D))).to(dtype)
    w = (rand(E, D) / D ** 0.5).to(dtype)
    idx = torch.topk(x.float() @ w.float().t(), k).indices.to(torch.int32) if k <= E else torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    mask = None
    if masked:
        mask = torch.arange(L, device="cuda") < torch.randint(0, L + 1, (S, 1), generator=g, device="cuda")
    return dict(x=x, w=w, idx=idx, S=S, mask=mask, alpha=0.3, dloss=torch.rand((), generator=g, device="cuda") + 0.5,
                dweight=(0.1 * rand(T, k)).to(dtype) if weights else None)


def call(p):
    from comfyui_amd import functional as HF
    loss, counts, scores = HF.gate_balance(p["x"], p["w"], p["idx"], alpha=p["alpha"], sequences=p["S"], mask=p["mask"])
    return (loss, counts, scores, *HF.gate_balance_backward(p["dloss"], p["x"], p["w"], p["idx"], counts, scores, alpha=p["alpha"], mask=p["mask"],
                                                            dweight=p["dweight"]))


def check(p):
    got = call(p)
    loss, counts, scores, dx, dw = router64.balance(p["x"], p["w"], p["idx"], p["alpha"], p["S"], p["mask"], p["dloss"], p["dweight"])
    assert got[1].dtype == torch.int32 and torch.equal(got[1].long(), counts)
    close(got[2], *scores, "scores")
    close(got[0], *loss, "loss")
    close(got[3], *dx, "dx")
    close(got[4], *dw, "dW")
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("S,L,D,E,k", [(1, 1, 8, 1, 1), (1, 1, 2560, 4, 2), (1, 64, 2560, 4, 2), (3, 5, 264, 3, 2), (2, 17, 520, 16, 4), (1, 63, 96, 16, 16),
                                       (8, 1, 128, 2, 1), (7, 100, 1000, 6, 2), (1, 333, 2048, 8, 2), (70, 9, 136, 5, 3), (300, 2, 64, 4, 2), (2, 640, 4096, 7, 2),
                                       (1, 16, 512, 2, 3)])
def test_sizes(dtype, masked, S, L, D, E, k):
    check(problem(S * 17 + L + D, S, L, D, E, k, dtype, masked))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,L,D,E,masked,weights", [(3, 1365, 2048, 8, True, True), (2, 6000, 2560, 4, False, False), (1, 20011, 328, 16, True, False),
                                                    (1, 8192, 640, 4, False, True)])
def test_many_tokens(dtype, S, L, D, E, masked, weights):
    check(problem(L, S, L, D, E, 2, dtype, masked, weights))


def test_masked_tokens_hold_anything():
    for dtype in TYPES:
        p = problem(3, 3, 90, 640, 4, 2, dtype, True)
        p["mask"][1] = False                                       # a sequence of padding
        p["mask"][0, 30:] = False
        clean = check(p)
        off = ~p["mask"].reshape(-1)
        p["x"][off] = float("nan")
        p["x"][off.nonzero()[3, 0]] = float("inf")
        p["idx"][off] = 77
        p["dweight"][off] = float("nan")
        dirty = call(p)
        for i in (0, 1, 3, 4):
            assert torch.equal(clean[i], dirty[i]), i
        assert torch.equal(clean[2][~off], dirty[2][~off]) and not dirty[3][off].any()
        p["mask"][:] = False                                       # nothing at all
        loss, counts, _, dx, dw = call(p)
        assert float(loss) == 0 and not counts.any() and not dx.any() and not dw.any()


def test_choices_out_of_range_and_twice():
    p = problem(4, 2, 50, 256, 5, 3, torch.bfloat16)
    p["idx"][::3, 0] = -1
    p["idx"][1::3, 1] = 5
    p["idx"][2::3, 2] = p["idx"][2::3, 0]
    p["idx"][7, 1] = 2 ** 31 - 1
    p["idx"][8, 1] = -2 ** 31
    check(p)


def test_the_gates_own_choices():
    """What gate_top2 chooses and returns beside it is what the gradients are of: its scores are these ones to the bf16 steps of logits and scores."""
    from comfyui_amd import functional as HF
    p = problem(6, 2, 500, 2560, 4, 2, torch.bfloat16)
    idx, weight = HF.gate_top2(p["x"], p["w"])
    p["idx"] = idx
    _, counts, scores, _, _ = check(p)
    assert int(counts.sum()) == 2 * 1000
    z = (p["x"].double() @ p["w"].double().t()).abs().amax(1, keepdim=True)
    near = torch.gather(scores.double(), 1, idx.long())
    assert ((weight.double() - near).abs() <= near * (2 * z * 2.0 ** -8 + 2.0 ** -8) * 1.1 + 1e-6).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_views_off_their_alignment(dtype):
    p = problem(8, 1, 77, 264, 4, 2, dtype)
    for k in ("x", "w", "idx", "dweight"):
        flat = torch.empty(p[k].numel() + 3, dtype=p[k].dtype, device="cuda")
        v = flat[3:].view(p[k].shape)
        v.copy_(p[k])
        p[k] = v
    check(p)


def test_large_logits():
    """Scores of 0 and 1: nothing overflows, and gradients are 0 where they are."""
    for dtype in TYPES:
        p = problem(2, 1, 40, 512, 6, 2, dtype)
        p["w"] = (p["w"].float() * 300).to(dtype)
        got = call(p)
        assert all(t.isfinite().all() for t in got)
        assert torch.equal(got[2].amax(1), torch.ones_like(got[2][:, 0])) or got[2].amax(1).min() > 0.5


def test_no_tokens():
    from comfyui_amd import functional as HF
    x, w = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16), torch.zeros((3, 64), device="cuda", dtype=torch.bfloat16)
    idx = torch.empty((0, 2), device="cuda", dtype=torch.int32)
    loss, counts, scores = HF.gate_balance(x, w, idx, sequences=2)
    assert float(loss) == 0 and counts.shape == (2, 3) and not counts.any() and scores.shape == (0, 3)
    dx, dw = HF.gate_balance_backward(torch.ones((), device="cuda"), x, w, idx, counts, scores)
    assert dx.shape == (0, 64) and not dw.any()


def test_refused_on_the_device():
    from comfyui_amd import functional as HF
    p = problem(1, 2, 4, 64, 4, 2, torch.bfloat16)
    x, w, idx = p["x"], p["w"], p["idx"]
    loss, counts, scores = HF.gate_balance(x, w, idx, sequences=2)
    one = torch.ones((), device="cuda")
    for bad in (lambda: HF.gate_balance(x[:, ::2], w, idx), lambda: HF.gate_balance(x, w[:, :32], idx), lambda: HF.gate_balance(x, w, idx[:4]),
                lambda: HF.gate_balance(x, w, idx, sequences=3), lambda: HF.gate_balance(x, w, idx, sequences=0), lambda: HF.gate_balance(x, w.cpu(), idx),
                lambda: HF.gate_balance(x, w, idx, mask=torch.ones(7, dtype=torch.bool, device="cuda")), lambda: HF.gate_balance(x[None], w, idx),
                lambda: HF.gate_balance_backward(one, x, w, idx, counts[:, :2], scores), lambda: HF.gate_balance_backward(one, x, w, idx, counts, scores.half()),
                lambda: HF.gate_balance_backward(one.double(), x, w, idx, counts, scores), lambda: HF.gate_balance_backward(one[None], x, w, idx, counts, scores),
                lambda: HF.gate_balance_backward(one, x, w, idx, counts, scores, dweight=p["dweight"].float())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: HF.gate_balance(x, w.half(), idx), lambda: HF.gate_balance(x, w, idx.long()),
                lambda: HF.gate_balance(x, w, idx, mask=torch.ones(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="E=17"):
        HF.gate_balance(x, torch.zeros((17, 64), device="cuda", dtype=torch.bfloat16), idx)
    with pytest.raises(RuntimeError, match="D=60"):
        HF.gate_balance(x[:, :60].contiguous(), w[:, :60].contiguous(), idx)


@pytest.mark.parametrize("S,L", [(1, 40), (2, 1500)])
def test_captured_replayed_and_on_another_stream(S, L):
    """Two graphs with workspaces of their own, replayed in turn with eager work between, on inputs and masks written anew."""
    sets = [problem(s, S, L, 1032, 5, 2, torch.bfloat16, masked=True) for s in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        elsewhere = [call(s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    for s, got in zip(sets, elsewhere):
        assert all(torch.equal(a, c) for a, c in zip(call(s), got))
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(s))
        graphs.append(graph)
    for turn in range(3):
        for i, s in enumerate(sets):
            new = problem(10 * turn + i + 5, S, L, 1032, 5, 2, torch.bfloat16, masked=True)
            for k in ("x", "w", "idx", "mask", "dloss", "dweight"):
                s[k].copy_(new[k])
        for graph in graphs:
            graph.replay()
        for s, out in zip(sets, outs):
            assert all(torch.equal(a, c) for a, c in zip(call(s), out)), turn
        torch.cuda.synchronize()
