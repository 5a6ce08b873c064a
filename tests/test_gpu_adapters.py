"""Adapters of many requests and their gradients against 64 bits (tests/adapters64.py derives the tolerances)."""
import pytest
import torch

from tests import adapters64
from tests.norm64 import close

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def problem(seed, requests, per, K, N, n, R, dtype, index=None):
    g = gen(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    T = requests * per
    channel = torch.exp(0.7 * rand(K))
    if index is None:
        index = torch.randint(-1, n, (requests,), generator=torch.Generator().manual_seed(seed))
    return dict(x=(rand(T, K) * channel).to(dtype), base=rand(T, N).to(dtype), dy=rand(T, N).to(dtype), a=(rand(n, R, K) / K ** 0.5).to(dtype),
                b=(rand(n, N, R) / R ** 0.5).to(dtype), scale=torch.rand(n, generator=g, device="cuda") + 0.5, index=index.to(torch.int32).cuda())


def check(p):
    from comfyui_amd import functional as HF
    out = HF.add_adapters(p["base"], p["x"], p["a"], p["b"], p["scale"], p["index"])
    close(out, *adapters64.forward(p["base"], p["x"], p["a"], p["b"], p["scale"], p["index"]), "out")
    check_backward(p)
    return out


def check_backward(p):
    from comfyui_amd import functional as HF
    got = HF.add_adapters_backward(p["dy"], p["x"], p["a"], p["b"], p["scale"], p["index"])
    for name, g, (want, err) in zip(("dx", "da", "db"), got, adapters64.backward(p["dy"], p["x"], p["a"], p["b"], p["scale"], p["index"])):
        close(g, want, err, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,per,K,N,n,R", [
    (1, 1, 64, 64, 1, 8), (1, 1, 2560, 6912, 4, 16), (1, 3, 8, 8, 2, 1), (5, 1, 100, 36, 3, 5), (16, 1, 256, 512, 16, 16), (17, 1, 264, 520, 9, 24),
    (48, 1, 6912, 2560, 40, 32), (7, 5, 1000, 328, 4, 40), (3, 33, 777, 333, 2, 7), (2, 64, 640, 1088, 3, 64), (2, 65, 512, 256, 2, 72), (1, 130, 1, 1, 1, 1),
    (4, 150, 320, 1100, 3, 128), (2, 300, 328, 136, 2, 136), (3, 257, 96, 640, 2, 256), (700, 1, 72, 88, 5, 16), (300, 2, 640, 264, 64, 8), (1, 600, 9, 2560, 2, 3)])
def test_sizes(dtype, requests, per, K, N, n, R):
    check(problem(requests * 31 + per + R, requests, per, K, N, n, R, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,per,K,N,n,R", [(3, 333, 2048, 8192, 2, 24), (2, 4096, 2560, 1280, 2, 32), (4, 1024, 640, 2560, 1, 64), (8, 700, 2560, 640, 8, 96)])
def test_many_rows(dtype, requests, per, K, N, n, R):
    check(problem(requests + per, requests, per, K, N, n, R, dtype))


def test_every_row_with_an_index_of_its_own_in_any_order():
    p = problem(1, 3000, 1, 264, 392, 7, 16, torch.bfloat16)
    check(p)
    p = problem(2, 2500, 1, 264, 392, 300, 8, torch.float16)
    check(p)


def test_rows_without_an_adapter_are_the_base_bit_for_bit():
    from comfyui_amd import functional as HF
    for per in (1, 100):
        index = torch.tensor([-1, 0, -7, 3, 2 ** 31 - 1, 1, -2 ** 31, 2])      # 3 and more: there are three
        p = problem(5, 8, per, 320, 200, 3, 16, torch.bfloat16, index)
        p["base"].view(torch.int16)[0, :4] = torch.tensor([0x7fc1, -1, -0x8000, 0x0001], dtype=torch.int16)   # NaN patterns, -0, a subnormal
        out = check_rows(p)
        none = ((index < 0) | (index > 2)).repeat_interleave(per).cuda()
        assert torch.equal(out.view(torch.int16)[none], p["base"].view(torch.int16)[none])
        dx, _, _ = HF.add_adapters_backward(p["dy"], p["x"], p["a"], p["b"], p["scale"], p["index"])
        assert not dx[none].any() and dx[~none].any()
        # nobody has an adapter
        p["index"].fill_(-1)
        assert torch.equal(HF.add_adapters(p["base"], p["x"], p["a"], p["b"], p["scale"], p["index"]).view(torch.int16), p["base"].view(torch.int16))
        assert not any(t.any() for t in HF.add_adapters_backward(p["dy"], p["x"], p["a"], p["b"], p["scale"], p["index"]))


def check_rows(p):
    from comfyui_amd import functional as HF
    out = HF.add_adapters(p["base"], p["x"], p["a"], p["b"], p["scale"], p["index"])
    want, err = adapters64.forward(p["base"].nan_to_num(), p["x"], p["a"], p["b"], p["scale"], p["index"])
    ok = p["base"].isfinite()
    close(out[ok], want[ok], err[ok], "out")
    return out


@pytest.mark.parametrize("per", [1, 9, 100])
def test_bad_values_of_one_request_reach_no_other(per):
    """NaN and infinities in rows, gradients and weights of one adapter."""
    from comfyui_amd import functional as HF
    for dtype in TYPES:
        p = problem(per, 12, per, 328, 456, 3, 24, dtype, torch.tensor([0, 1, 2, -1] * 3))
        of = p["index"].repeat_interleave(per)
        good = (of == 0) | (of == 2)
        names = ("x", "a", "b", "scale", "index")
        clean = HF.add_adapters(p["base"], *(p[k] for k in names)), *HF.add_adapters_backward(p["dy"], *(p[k] for k in names))
        for i, bad in enumerate((float("nan"), float("inf"), float("-inf"))):
            p["x"][~good, 7 + i] = bad
            p["dy"][~good, 3 + i] = bad
            p["a"][1, i, 11] = bad
            p["b"][1, 5, i] = bad
        p["scale"][1] = float("nan")
        out, dx, da, db = HF.add_adapters(p["base"], *(p[k] for k in names)), *HF.add_adapters_backward(p["dy"], *(p[k] for k in names))
        for got, want in ((out, clean[0]), (dx, clean[1])):
            assert torch.equal(got[good], want[good])
            assert got[of == 1].isnan().any()
        for got, want in ((da, clean[2]), (db, clean[3])):
            assert torch.equal(got[[0, 2]], want[[0, 2]]) and got[1].isnan().all()


def test_the_same_request_twice_and_in_place():
    from comfyui_amd import functional as HF
    p = problem(9, 6, 40, 512, 640, 2, 16, torch.bfloat16, torch.tensor([1, 1, 0, 1, -1, 1]))
    p["x"][40:80] = p["x"][:40]
    p["base"][40:80] = p["base"][:40]
    out = check(p)
    assert torch.equal(out[:40], out[40:80])
    base = p["base"].clone()
    back = HF.add_adapters(base, p["x"], p["a"], p["b"], p["scale"], p["index"], out=base)
    assert back is base and torch.equal(base, out)
    shaped = HF.add_adapters(p["base"].view(6, 40, 640), p["x"].view(6, 40, 512), p["a"], p["b"], p["scale"], p["index"])
    assert shaped.shape == (6, 40, 640) and torch.equal(shaped.view(-1, 640), out)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_off_their_alignment(dtype):
    p = problem(4, 3, 41, 168, 136, 2, 24, dtype)

    def shifted(t):
        flat = torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")
        v = flat[3:].view(t.shape)
        v.copy_(t)
        return v

    check({k: shifted(v) for k, v in p.items()})


def test_values_of_very_different_size():
    """Gradients as small as a loss scale of 1 leaves them, and as large as fp16 holds: the narrow values are fp32."""
    for dtype in TYPES:
        for factor in (2.0 ** -20, 2.0 ** 12):
            p = problem(8, 2, 70, 512, 640, 2, 16, dtype)
            p["dy"] = (p["dy"].float() * factor).to(dtype)
            p["a"], p["b"] = (p["a"].float() * 0.25).to(dtype), (p["b"].float() * (8.0 if factor < 1 else 0.01)).to(dtype)
            p["x"] = (p["x"].float() * (64.0 if factor < 1 else 2.0 ** -8)).to(dtype)
            check_backward(p)


def test_no_rows():
    from comfyui_amd import functional as HF
    p = problem(1, 2, 3, 64, 32, 2, 8, torch.bfloat16)
    x, base, index = p["x"][:0], p["base"][:0], p["index"][:0]
    assert HF.add_adapters(base, x, p["a"], p["b"], p["scale"], index).shape == (0, 32)
    dx, da, db = HF.add_adapters_backward(base, x, p["a"], p["b"], p["scale"], index)
    assert dx.shape == (0, 64) and not da.any() and not db.any() and da.shape == p["a"].shape and db.shape == p["b"].shape


def test_refused_on_the_device():
    from comfyui_amd import functional as HF
    p = problem(1, 4, 2, 64, 32, 2, 8, torch.bfloat16)
    names = ("base", "x", "a", "b", "scale", "index")

    def call(**kw):
        return HF.add_adapters(*({**p, **kw}[k] for k in names), out=kw.get("out"))

    for bad in (dict(base=p["base"][:4]), dict(base=p["base"].t().contiguous()), dict(x=p["x"][:, :32]), dict(x=p["x"][:, ::2]), dict(a=p["a"][:1]),
                dict(b=p["b"][:, :, :4]), dict(scale=p["scale"][:1]), dict(index=p["index"][:3]), dict(index=p["index"].cpu()), dict(index=p["index"][:0]),
                dict(out=p["base"][:2]), dict(x=p["x"][0]), dict(a=p["a"][0]), dict(a=p["a"].transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(base=p["base"].half(), x=p["x"].half()), dict(scale=p["scale"].double()), dict(index=p["index"].long())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(ValueError):
        HF.add_adapters_backward(p["dy"][:4], *(p[k] for k in names[1:]))
    big = dict(a=torch.zeros((1, 257, 64), device="cuda", dtype=torch.bfloat16), b=torch.zeros((1, 32, 257), device="cuda", dtype=torch.bfloat16), scale=p["scale"][:1])
    with pytest.raises(RuntimeError, match="257"):
        call(**big)


@pytest.mark.parametrize("requests,per", [(8, 1), (3, 200)])
def test_captured_replayed_and_on_another_stream(requests, per):
    """Two graphs with workspaces of their own, replayed in turn with eager work between, on inputs and indices written anew."""
    from comfyui_amd import functional as HF
    sets = [problem(s, requests, per, 640, 1032, 3, 16, torch.bfloat16) for s in (1, 2)]
    names = ("x", "a", "b", "scale", "index")

    def call(p):
        return (HF.add_adapters(p["base"], *(p[k] for k in names)), *HF.add_adapters_backward(p["dy"], *(p[k] for k in names)))

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
            new = problem(10 * turn + i + 5, requests, per, 640, 1032, 3, 16, torch.bfloat16)
            for k in new:
                s[k].copy_(new[k])
        for graph in graphs:
            graph.replay()
        for s, out in zip(sets, outs):
            assert all(torch.equal(a, c) for a, c in zip(call(s), out)), turn
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,per,K,N,n,R,used", [(3, 700, 264, 520, 40, 16, (7, 39)), (2, 3000, 136, 648, 300, 24, (299,)), (600, 1, 328, 264, 30, 72, None),
                                                       (70, 15, 264, 776, 9, 100, None), (70, 16, 264, 776, 9, 33, None), (5, 1, 96, 72, 4096, 8, (0, 31, 32, 4095)),
                                                       (900, 2, 72, 1032, 700, 8, None), (2, 1500, 1032, 72, 33, 96, (32, 1))])
def test_many_adapters_of_which_few_are_used(dtype, requests, per, K, N, n, R, used):
    """Rows dealt to blocks by runs, each with whatever adapters it has: all rows of one, a run with hundreds, most without any rows."""
    index = None
    if used is not None:
        index = torch.tensor(used)[torch.randint(0, len(used), (requests,), generator=torch.Generator().manual_seed(n))]
    check(problem(n + R, requests, per, K, N, n, R, dtype, index))


@pytest.mark.parametrize("R", [65, 96, 128, 200])
def test_long_ranks_over_runs_of_every_length(R):
    for rows in (511, 513, 560, 1000):
        check(problem(R + rows, 1, rows, 200, 392, 1, R, torch.bfloat16 if R % 2 else torch.float16, torch.tensor([0])))


@pytest.mark.parametrize("n,R", [(2048, 16), (2048, 40)])
def test_parts_that_are_too_many_to_be_cut_as_finely(n, R):
    """Adapters whose gradients, times the runs that the rows alone would be cut into, pass what the parts may take."""
    check(problem(n + R, 2, 1500, 72, 1032, n, R, torch.bfloat16, torch.tensor([5, n - 1])))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,N", [(120, 128), (129, 255), (136, 1160), (1025, 511), (2048, 640)])
def test_columns_that_end_inside_a_wave(dtype, K, N):
    """Waves that have the last 128 columns over again, or too few columns for that: short and long ranks, one adapter and rows of many."""
    for requests, per, n, R in ((2, 300, 2, 40), (1, 900, 1, 88), (1, 600, 1, 256), (40, 1, 5, 104), (3, 50, 2, 72)):
        check(problem(K + N + R, requests, per, K, N, n, R, dtype, None))
