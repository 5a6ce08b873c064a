"""The compiled calls of the layer norm, the balance loss and the adapters: they make the ordinary calls, and give the bytes that the same calls from Python give."""
import pytest
import torch

from tests import test_gpu_adapters, test_gpu_norm, test_gpu_router

pytestmark = pytest.mark.gpu


class Watched:
    def __init__(self, module):
        self.module, self.made = module, []

    def __getattr__(self, name):
        def call(*args):
            r = getattr(self.module, name)(*args)
            self.made.append((name, r is not None))
            return r
        return call


def calls():
    from comfyui_amd import functional as HF
    g = test_gpu_norm.gen(1)
    x = test_gpu_norm.rows_of(g, (3, 40, 328), torch.bfloat16)
    dy = torch.randn(x.shape, generator=g, device="cuda").bfloat16()
    w, b = test_gpu_norm.gains(g, 328, torch.float32)
    x2, dy2, scale = x.view(-1, 328), dy.view(-1, 328), test_gpu_norm.rows_of(g, (3, 1, 328), torch.bfloat16)
    yield "layer_norm", lambda: HF.layer_norm(x, w, b)
    yield "layer_norm", lambda: HF.layer_norm(x)
    yield "layer_norm_backward", lambda: HF.layer_norm_backward(dy, x, w, b)
    yield "layer_norm_backward", lambda: HF.layer_norm_backward(dy, x, w, b, gains=False)
    yield "layer_norm_backward", lambda: HF.layer_norm_backward(dy, x, bias=b)
    yield "ln_modulate_backward", lambda: HF.ln_modulate_backward(dy2, x2, scale[:, 0], 40)
    r = test_gpu_router.problem(2, 3, 50, 264, 5, 2, torch.float16, True)
    yield "gate_balance", lambda: HF.gate_balance(r["x"], r["w"], r["idx"], sequences=3, mask=r["mask"])
    yield "gate_balance", lambda: HF.gate_balance(r["x"], r["w"], r["idx"])
    loss, counts, scores = HF.gate_balance(r["x"], r["w"], r["idx"], sequences=3)
    for dweight in (None, r["dweight"]):
        yield "gate_balance_backward", lambda d=dweight: HF.gate_balance_backward(r["dloss"], r["x"], r["w"], r["idx"], counts, scores, mask=r["mask"], dweight=d)
    for per in (1, 30, 300):
        p = test_gpu_adapters.problem(3, 3, per, 264, 392, 2, 12, torch.bfloat16)
        rest = [p[k] for k in ("x", "a", "b", "scale", "index")]
        yield "add_adapters", lambda p=p, rest=rest: HF.add_adapters(p["base"], *rest)
        yield "add_adapters", lambda p=p, rest=rest: HF.add_adapters(p["base"], *rest, out=torch.empty_like(p["base"]))
        yield "add_adapters_backward", lambda p=p, rest=rest: HF.add_adapters_backward(p["dy"], *rest)


def test_the_same_bytes_with_and_without(monkeypatch):
    from comfyui_amd import functional as HF
    assert HF._row_calls is not None
    watched = Watched(HF._row_calls)
    for name, call in calls():
        monkeypatch.setattr(HF, "_row_calls", watched)
        watched.made.clear()
        with_it = call()
        assert watched.made == [(name, True)], (name, watched.made)
        monkeypatch.setattr(HF, "_row_calls", None)
        without = call()
        for a, b in zip(*(r if isinstance(r, tuple) else (r,) for r in (with_it, without))):
            assert (a is None) == (b is None) and (a is None or (a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b))), name


@pytest.mark.parametrize("tests", [test_gpu_norm, test_gpu_adapters, test_gpu_router])
def test_the_same_refusals_without(tests, monkeypatch):
    from comfyui_amd import functional as HF
    monkeypatch.setattr(HF, "_row_calls", None)
    tests.test_refused_on_the_device()


def test_out_is_returned_as_it_was_given():
    from comfyui_amd import functional as HF
    p = test_gpu_adapters.problem(4, 2, 5, 64, 40, 1, 8, torch.float16)
    out = torch.empty_like(p["base"])
    assert HF.add_adapters(p["base"], p["x"], p["a"], p["b"], p["scale"], p["index"], out=out) is out


def test_an_ordinary_call_makes_no_other_thread_wait():
    """Two threads with streams of their own: results as in one."""
    import threading
    from comfyui_amd import functional as HF
    p = test_gpu_adapters.problem(5, 3, 200, 640, 640, 2, 16, torch.bfloat16)
    rest = [p[k] for k in ("x", "a", "b", "scale", "index")]
    want = HF.add_adapters_backward(p["dy"], *rest)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i] = HF.add_adapters_backward(p["dy"], *rest)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want))
