"""Which way the modules take for Linears with a scale for each block of 128: decisions of the host, no device."""
import torch

from comfyui_amd import hidream, ops

FP8 = torch.float8_e4m3fn


def feed_forward(**kwargs):
    return hidream.FeedForwardSwiGLU(64, 96, operations=ops.block_fp8_ops, multiple_of=16, **kwargs)


def test_weights_turned_into_16_bits_do_not_lose_their_scales():
    """The kernels for plain 16-bit weights know no scales: a module cast as a whole is left to its Linears, which refuse it."""
    f = feed_forward().to(torch.bfloat16)
    assert f.w1.weight.dtype == torch.bfloat16 and f.w1.scale_weight is not None
    assert hidream._fusable_dtype([f]) is None
    assert hidream._fusable_dtype([feed_forward()]) is None
    plain = hidream.FeedForwardSwiGLU(64, 96, multiple_of=16, dtype=torch.bfloat16)
    assert hidream._fusable_dtype([plain]) == torch.bfloat16
    assert hidream._fusable_dtype([plain, f]) is None


class Other(torch.nn.Module):
    """An expert of somebody else's."""

    def __init__(self):
        super().__init__()
        self.up = torch.nn.Linear(64, 64, bias=False)

    def forward(self, x):
        return self.up(x)


def test_experts_of_another_class_are_asked_for_no_linears():
    """They are called as they are, with renormalised gate weights for one."""
    x = torch.zeros((1, 64), dtype=torch.bfloat16)
    assert hidream._block_parts([Other(), Other(), feed_forward()], x) is None
    assert hidream._block_parts([feed_forward(), Other()], x) is None


def test_weights_are_brought_over_only_where_they_are_used(monkeypatch):
    """Offloaded weights of feed-forwards whose gate/up has a bias, or that hold a Linear of another kind, are not moved or cast in vain."""
    moved = []
    parts = ops.block_fp8_ops.Linear.parts
    monkeypatch.setattr(ops.block_fp8_ops.Linear, "parts", lambda self, x: moved.append(self) or parts(self, x))
    x = torch.zeros((1, 64), dtype=torch.bfloat16)
    plain, biased, mixed = feed_forward(), feed_forward(), feed_forward()
    assert hidream._block_parts([plain, plain], x) is not None and len(moved) == 6
    del moved[:]
    biased.w3.bias = torch.nn.Parameter(torch.zeros(96, dtype=torch.bfloat16))
    mixed.w2 = ops.manual_cast.Linear(96, 64, bias=False)
    assert hidream._block_parts([plain, biased], x) is None and hidream._block_parts([plain, mixed], x) is None
    assert moved == []
    down = feed_forward()
    down.w2.bias = torch.nn.Parameter(torch.zeros(64, dtype=torch.bfloat16))
    assert hidream._block_parts([plain, down], x)[1][1][2] is not None


def test_a_linear_wrapped_in_another_module_is_left_to_itself():
    """Wrappers (adapters) need not have a bias to be looked at."""
    x = torch.zeros((1, 64), dtype=torch.bfloat16)
    plain, wrapped = feed_forward(), feed_forward()
    wrapped.w1 = torch.nn.Sequential(wrapped.w1)
    assert hidream._block_parts([plain, wrapped], x) is None
