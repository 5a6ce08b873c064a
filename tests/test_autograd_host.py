"""What the differentiable functions and the modules around them refuse or decide without a device."""
import pytest
import torch

BF16 = torch.bfloat16


def test_inputs_with_gradients_are_refused_while_a_graph_is_captured(monkeypatch):
    from comfyui_amd import autograd as A
    x = torch.zeros((4, 16), dtype=BF16, requires_grad=True)
    w = torch.zeros((3, 16), dtype=BF16)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    a, b = torch.zeros((1, 8, 16), dtype=BF16), torch.zeros((1, 16, 8), dtype=BF16)
    for call in (lambda: A.layer_norm(x), lambda: A.ln_modulate(x, x[:1], x[:1], 4), lambda: A.gate(x, w),
                 lambda: A.add_adapters(x, x, a, b, torch.ones(1), torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="while a graph is captured"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):      # without gradients it is an ordinary call
            call()


def test_a_captured_backward_pass_of_an_eager_call_is_refused(monkeypatch):
    from comfyui_amd import autograd as A
    from comfyui_amd import functional as HF
    like = lambda x, *a: x.clone()  # noqa: E731
    monkeypatch.setattr(HF, "layer_norm", like)
    monkeypatch.setattr(HF, "ln_modulate", like)
    monkeypatch.setattr(HF, "add_adapters", like)
    monkeypatch.setattr(HF, "gate_top2", lambda x, w: (torch.zeros((4, 2), dtype=torch.int32), x[:, :2].clone()))
    monkeypatch.setattr(HF, "gate_balance", lambda *a: (torch.zeros(()), torch.zeros((1, 3), dtype=torch.int32), torch.zeros((4, 3))))
    x = torch.zeros((4, 16), dtype=BF16, requires_grad=True)
    a, b = torch.zeros((1, 8, 16), dtype=BF16), torch.zeros((1, 16, 8), dtype=BF16)
    results = [A.layer_norm(x), A.ln_modulate(x, x[:1], x[:1], 4), A.gate(x, torch.zeros((3, 16), dtype=BF16))[2],
               A.add_adapters(x, x, a, b, torch.ones(1), torch.zeros(1, dtype=torch.int32))]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for y in results:
        with pytest.raises(RuntimeError, match="while a graph is captured"):
            y.sum().backward()


def test_scales_have_no_gradient():
    from comfyui_amd import autograd as A
    x = torch.zeros((4, 16), dtype=BF16)
    a, b = torch.zeros((1, 8, 16), dtype=BF16), torch.zeros((1, 16, 8), dtype=BF16)
    with pytest.raises(RuntimeError, match="scales"):
        A.add_adapters(x, x, a, b, torch.ones(1, requires_grad=True), torch.zeros(1, dtype=torch.int32))


def test_layer_norm_module_keeps_the_names_and_refuses_other_axes():
    from comfyui_amd import ops
    for cls in (ops.disable_weight_init, ops.manual_cast, ops.fp8_ops, ops.block_fp8_ops, ops.scaled_fp8_ops()):
        m = cls.LayerNorm(16, dtype=BF16)
        assert set(m.state_dict()) == {"weight", "bias"} and isinstance(m, torch.nn.LayerNorm)
        with pytest.raises(RuntimeError, match="no CPU path"):
            m(torch.zeros((2, 16), dtype=BF16))
    assert ops.manual_cast.LayerNorm.comfy_cast_weights and not ops.disable_weight_init.LayerNorm.comfy_cast_weights
    with pytest.raises(NotImplementedError):
        ops.disable_weight_init.LayerNorm((4, 16))(torch.zeros((2, 4, 16)))
    with pytest.raises(ValueError):
        ops.disable_weight_init.LayerNorm(16)(torch.zeros((2, 8)))


def test_adapters_of_different_ranks_are_filled_up():
    from comfyui_amd import ops
    g = torch.Generator().manual_seed(1)
    parts = [(torch.randn((r, 12), generator=g), torch.randn((10, r), generator=g), s) for r, s in ((4, 0.5), (9, 2.0), (1, 1.0))]
    ad = ops.Adapters.stack(parts, dtype=BF16)
    assert ad.a.shape == (3, 9, 12) and ad.b.shape == (3, 10, 9) and ad.scale.tolist() == [0.5, 2.0, 1.0] and ad.a.dtype == BF16
    for i, (a, b, _) in enumerate(parts):
        assert torch.equal(ad.a[i, :a.shape[0]], a.to(BF16)) and not ad.a[i, a.shape[0]:].any()
        assert torch.equal(ad.b[i, :, :a.shape[0]], b.to(BF16)) and not ad.b[i, :, a.shape[0]:].any()


def test_linears_with_adapters_are_called_by_themselves():
    """No fused path takes a Linear with adapters, cached structures or not, and the other Linears are as before."""
    from comfyui_amd import hidream, hunyuan3d, ops
    ff = hidream.FeedForwardSwiGLU(128, 384, dtype=BF16)
    assert hidream._fusable_dtype([ff]) == BF16 and hidream._pack_key([ff], torch.device("cpu")) is not None
    ad = ops.Adapters.stack([(torch.zeros((8, 128)), torch.zeros((256, 8)), 1.0)], dtype=BF16)
    ff.w3.adapters = ad
    assert ops.adapters_of(ff.w3) is ad and ops.adapters_of(ff.w1) is None
    assert hidream._fusable_dtype([ff]) is None and hidream._pack_key([ff], torch.device("cpu")) is None
    x = torch.zeros((2, 128), dtype=BF16)
    block = ops.block_fp8_ops.Linear(128, 256, bias=False)
    assert ops.block_fp8_parts([block], x) is not None
    block.adapters = ad
    assert ops.block_fp8_parts([block], x) is None
    lin = torch.nn.Linear(128, 256, dtype=BF16)
    assert hunyuan3d._plain_pair(lin, x) is not None
    lin.adapters = ad
    assert hunyuan3d._plain_pair(lin, x) is None
    del ff.w3.adapters
    assert hidream._fusable_dtype([ff]) == BF16


def test_adapters_want_an_index_and_no_gradients():
    from comfyui_amd import ops
    ad = ops.Adapters.stack([(torch.zeros((8, 16)), torch.zeros((16, 8)), 1.0)], dtype=BF16)
    x = torch.zeros((4, 16), dtype=BF16)
    with pytest.raises(RuntimeError, match="index"):
        ad(x, x)
    ad.a.requires_grad_()
    with pytest.raises(RuntimeError, match="inference only"):
        ad(x, x)
    ad.a.requires_grad_(False)
    ad.index = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="divide"), ops.routed_adapters(torch.nn.ModuleList([_holder(ad)]), 4, torch.arange(4)):
        pass
    ad.index = torch.tensor([5, 7], dtype=torch.int32)
    with ops.routed_adapters(_holder(ad), 4, torch.tensor([7, 0, 3, 4], dtype=torch.int32)):
        assert ad._rows.tolist() == [7, 5, 5, 7]          # tokens 3, 0, 1, 2 of two requests of two
    assert ad._rows is None


def _holder(ad):
    lin = torch.nn.Linear(16, 16)
    lin.adapters = ad
    return lin


def test_route_refuses_what_has_no_gradient():
    from comfyui_amd import hidream, hunyuan3d
    g = hidream.MoEGate(16, dtype=BF16)
    g.norm_topk_prob = True
    with pytest.raises(NotImplementedError):
        g.route(torch.zeros((1, 2, 16), dtype=BF16))
    with pytest.raises(NotImplementedError):
        hunyuan3d.MoEGate(16, num_experts_per_tok=3, dtype=BF16).route(torch.zeros((1, 2, 16), dtype=BF16))
