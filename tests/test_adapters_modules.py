"""Adapters beside a Linear as a module: hooks, `forward` called by itself, subclasses and other operations classes. The device's calls are stood in for by
their formulas."""
import pytest
import torch

from comfyui_amd import functional as HF
from comfyui_amd import hidream, hunyuan3d, ops

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    def add_adapters(base, x, a, b, scale, index, **kwargs):
        assert x.dim() >= 2 and base.shape[:-1] == x.shape[:-1]
        out = base.clone().reshape(-1, base.shape[-1])
        per = x.numel() // x.shape[-1] // index.numel()
        for t, row in enumerate(x.reshape(-1, x.shape[-1])):
            i = int(index[t // per])
            if 0 <= i < a.shape[0]:
                out[t] += scale[i].to(out.dtype) * (b[i] @ (a[i] @ row))
        return out.view(base.shape)

    monkeypatch.setattr(HF, "linear", lambda x, w, *a, bias=None, **k: torch.nn.functional.linear(x, w.to(x.dtype), bias))
    monkeypatch.setattr(HF, "add_adapters", add_adapters)
    monkeypatch.setattr(HF, "silu_mul", lambda a, b: torch.nn.functional.silu(a) * b)
    monkeypatch.setattr(HF, "gelu", torch.nn.functional.gelu)


def identity(cls=ops.disable_weight_init.Linear, n=16):
    """A Linear and adapters that both give their input back."""
    lin = cls(n, n, bias=False, dtype=torch.float32)
    with torch.no_grad():
        lin.weight.copy_(torch.eye(n))
    lin.adapters = ops.Adapters(torch.eye(n)[None], torch.eye(n)[None], torch.ones(1))
    lin.adapters.index = torch.zeros(1, dtype=torch.int32)
    return lin


ONE = torch.ones((2, 16))


@pytest.mark.parametrize("cls", [ops.disable_weight_init.Linear, ops.manual_cast.Linear])
def test_hooks(cls):
    lin = identity(cls)
    with torch.no_grad():
        assert torch.equal(lin(ONE), 2 * ONE)
        first = lin.register_forward_pre_hook(lambda m, args: (args[0] * 10,))
        assert torch.equal(lin(ONE), 20 * ONE)
        seen = []
        second = lin.register_forward_hook(lambda m, args, out: seen.append(out) or out + 1)
        assert torch.equal(lin(ONE), 21 * ONE) and torch.equal(seen[0], 20 * ONE)
        first.remove(), second.remove()
        del lin.adapters
        assert torch.equal(lin(ONE), ONE)


def test_forward_by_itself_and_the_classes_own():
    lin = identity()
    with torch.no_grad():
        assert torch.equal(lin.forward(ONE), 2 * ONE) and torch.equal(lin(input=ONE), 2 * ONE) and torch.equal(lin.forward(input=ONE), 2 * ONE)
        assert torch.equal(type(lin).forward(lin, ONE), ONE)      # the product alone
        own = lin.forward                                          # as a wrapper holds it
        lin.forward = lambda x: own(x) + 1
        assert torch.equal(lin(ONE), 3 * ONE)
        del lin.adapters
        assert torch.equal(lin(ONE), 2 * ONE)
        del lin.forward
        assert torch.equal(lin(input=ONE), ONE)
    assert ops.manual_cast.Linear.forward is ops.disable_weight_init.Linear.forward is ops.block_fp8_ops.Linear.forward


def test_subclasses():
    class Twice(ops.disable_weight_init.Linear):
        def forward(self, x):
            return super().forward(x) * 2

    class Own(ops.disable_weight_init.Linear):
        def forward(self, x):
            return x * 5

    class Mixin:
        def forward(self, x):
            return super().forward(x) * 2

    class Mixed(Mixin, ops.manual_cast.Linear):
        pass

    with torch.no_grad():
        assert torch.equal(identity(Mixed)(ONE), 3 * ONE) and torch.equal(identity(Twice)(x=ONE), 3 * ONE)
        assert torch.equal(identity(Twice)(ONE), 3 * ONE)          # they join the outer result
        assert torch.equal(identity(Twice)(input=ONE), 3 * ONE)
        assert torch.equal(identity(Own)(ONE), 6 * ONE) and torch.equal(identity(Own).forward(ONE), 6 * ONE)
        lin = identity(Twice)
        lin.adapters.index = None
        for _ in range(2):                                          # an error leaves nothing behind
            with pytest.raises(RuntimeError, match="index"):
                lin(ONE)
        lin.adapters.index = torch.zeros(1, dtype=torch.int32)
        assert torch.equal(lin(ONE), 3 * ONE)


def test_a_replaced_forward_that_leaves_them_out_is_refused(monkeypatch):
    lin = identity()
    lin.forward = lambda x: x
    with torch.no_grad(), pytest.raises(RuntimeError, match="leaves them out"):
        lin(ONE)
    other = identity()
    own = ops.disable_weight_init.Linear.forward
    monkeypatch.setattr(ops.disable_weight_init.Linear, "forward", lambda self, x: own(self, x))
    with torch.no_grad(), pytest.raises(RuntimeError, match="leaves them out"):
        other(ONE)


class Joins(torch.nn.Linear):
    """Another class that knows what to do with them."""

    def forward(self, x):
        return self.adapters(super().forward(x), x) if hasattr(self, "adapters") else super().forward(x)


def test_linears_of_other_classes():
    class operations:
        Linear = torch.nn.Linear

    class joining:
        Linear = Joins

    def adapters(lin):
        ad = ops.Adapters(torch.ones((1, 2, lin.in_features)), torch.ones((1, lin.out_features, 2)), torch.ones(1))
        ad.index = torch.zeros(1, dtype=torch.int32)
        return ad

    x = torch.ones((3, 16))
    for at in ("w1", "w2", "w3"):
        with torch.no_grad():
            ff = hidream.FeedForwardSwiGLU(16, 32, multiple_of=16, dtype=torch.float32, operations=operations)
            before = ff(x)
            lin = getattr(ff, at)
            lin.adapters = adapters(lin)
            with pytest.raises(RuntimeError, match="torch.nn.modules.linear.Linear whose forward leaves them out"):
                ff(x)
            del lin.adapters
            assert torch.equal(ff(x), before)
            ff = hidream.FeedForwardSwiGLU(16, 32, multiple_of=16, dtype=torch.float32, operations=joining)
            before = ff(x)
            lin = getattr(ff, at)
            lin.adapters = adapters(lin)
            assert not torch.equal(ff(x), before)
    lin = torch.nn.Linear(16, 16)
    lin.adapters = torch.nn.ModuleDict()                # a name of its own
    assert torch.equal(ops.call_linear(lin, ONE), lin(ONE))
    with ops.routed_adapters(torch.nn.ModuleList([lin]), 4, torch.arange(8)):
        pass


def test_linears_of_other_classes_in_hunyuan3d(monkeypatch):
    monkeypatch.setattr(hunyuan3d, "_need", lambda x: None)

    class operations:
        Linear = torch.nn.Linear

    x = torch.ones((3, 16))
    with torch.no_grad():
        ff = hunyuan3d.FeedForward(16, inner_dim=32, operations=operations, dtype=torch.float32)
        for lin in (ff.net[0].proj, ff.net[2]):
            lin.adapters = ops.Adapters(torch.ones((1, 2, lin.in_features)), torch.ones((1, lin.out_features, 2)), torch.ones(1))
            lin.adapters.index = torch.zeros(1, dtype=torch.int32)
            monkeypatch.setattr(hunyuan3d, "_plain_pair", lambda lin, x: None)
            with pytest.raises(RuntimeError, match="leaves them out"):
                ff(x)
            del lin.adapters
        assert ff(x).shape == (3, 16)


def test_a_cast_of_the_model_leaves_the_scales_fp32():
    scale = torch.tensor([0.1, 1.0 / 3.0])
    ad = ops.Adapters(torch.ones((2, 4, 16)), torch.ones((2, 16, 4)), scale.clone())
    lin = identity()
    lin.adapters = ad
    for cast in (lambda m: m.to(BF16), lambda m: m.half(), lambda m: m.to(torch.device("cpu"), torch.bfloat16), lambda m: m.bfloat16().float()):
        cast(lin)
        assert ad.scale.dtype == torch.float32 and torch.equal(ad.scale, scale) and ad.a.dtype == lin.weight.dtype and "scale" in ad.state_dict()
    lin.to(BF16)
    with torch.no_grad():
        ad.index = torch.ones(1, dtype=torch.int32)
        assert lin(ONE.to(BF16)).isfinite().all()
    lin.to("meta")
    assert ad.scale.device.type == "meta" and ad.scale.dtype == torch.float32
    lin.to(torch.float16).to_empty(device="cpu")
    assert ad.scale.device.type == "cpu" and ad.scale.dtype == torch.float32


def test_routed_rows_of_all_adapters_or_none():
    first, second = identity(), identity()
    first.adapters.index = torch.tensor([0, -1], dtype=torch.int32)
    for bad in (None, torch.zeros(3, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)):
        second.adapters.index = bad
        with pytest.raises(RuntimeError, match="index"), ops.routed_adapters(torch.nn.ModuleList([first, second]), 4, torch.tensor([7, 0])):
            pass
        assert first.adapters._rows is None and second.adapters._rows is None
    with torch.no_grad():
        assert torch.equal(first(ONE), torch.cat([2 * ONE[:1], ONE[1:]]))       # by `index`, not by rows of an earlier call
    second.adapters.index = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(IndexError), ops.routed_adapters(torch.nn.ModuleList([first, second]), 4, torch.tensor([7, 800])):
        pass
    assert first.adapters._rows is None
    with ops.routed_adapters(torch.nn.ModuleList([first, second]), 4, torch.tensor([7, 0])):
        assert first.adapters._rows.tolist() == [-1, 0] and second.adapters._rows.tolist() == [0, 0]
    assert first.adapters._rows is None and second.adapters._rows is None


def test_a_single_row_without_an_axis_of_its_own():
    lin = identity()
    with torch.no_grad():
        y = lin(ONE[0])
    assert y.shape == (16,) and torch.equal(y, 2 * ONE[0])
