"""ops.LayerNorm's ways to be called, without a device: it gets as far as the refusal of a CPU tensor, or to the call that it stands for."""
import pytest
import torch

from comfyui_amd import autograd, ops


@pytest.mark.parametrize("cls", [ops.disable_weight_init, ops.manual_cast])
def test_input_by_name(cls, monkeypatch):
    m = cls.LayerNorm(16, dtype=torch.bfloat16)
    x = torch.zeros((2, 16), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        m(input=x)
    monkeypatch.setattr(autograd, "layer_norm", lambda x, w, b, eps: (x, w, b, eps))
    by_name, by_place = m(input=x), m(x)
    assert by_name[0] is by_place[0] is x and torch.equal(by_name[1], m.weight) and by_name[3] == 1e-5


@pytest.mark.parametrize("cls", [ops.disable_weight_init, ops.manual_cast])
def test_without_a_bias_and_with_functions(cls, monkeypatch):
    monkeypatch.setattr(autograd, "layer_norm", lambda x, w, b, eps: (x, w, b, eps))
    m = cls.LayerNorm(16, bias=False, dtype=torch.bfloat16)
    with torch.no_grad():
        m.weight.fill_(2)
    x = torch.zeros((2, 16), dtype=torch.bfloat16)
    assert m(x)[2] is None and m(x)[1].eq(2).all()
    m.weight_function = [lambda w: w + 1]
    assert m(x)[1].eq(3).all() and m.weight.eq(2).all()
