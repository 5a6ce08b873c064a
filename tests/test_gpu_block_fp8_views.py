"""Activations that are views starting anywhere in their storage, through the modules on weights with block scales: as the other modules take them."""
import pytest
import torch

from tests.test_gpu_block_fp8_layers import layer

pytestmark = pytest.mark.gpu


def shifted(x):
    """x's values in a storage that starts one element early."""
    v = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
    assert v.copy_(x).data_ptr() % 16 != 0 and v.is_contiguous()
    return v


@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_linear_feed_forward_and_layer(tokens):
    m, g, synth = layer()
    x = synth.make_input(g, tokens, dim=512).cuda()
    for f in (m.experts[0].w1, m.experts[0], m):
        assert torch.equal(f(shifted(x)), f(x))
    shift, scale, gate = (torch.randn((1, 1, 512), generator=g).bfloat16().cuda() for _ in range(3))
    assert torch.equal(m.forward_branch(shifted(x), shift, scale, gate), m.forward_branch(x, shift, scale, gate))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_hunyuan_block(dtype):
    from comfyui_amd import hunyuan3d, ops
    torch.manual_seed(5)
    b = hunyuan3d.MoEBlock(256, num_experts=4, ff_inner_dim=528, operations=ops.block_fp8_ops, device="cuda", dtype=dtype).eval()
    with torch.no_grad():
        for name, p in b.state_dict().items():
            if name.endswith("scale_weight"):
                p.fill_(2.0 ** -9)
            else:
                p.copy_(torch.randn(p.shape, device="cuda") * (40 if p.dtype == torch.float8_e4m3fn else 0.05))
    x = torch.randn((1, 30, 256), device="cuda").to(dtype)
    y = b(x)
    assert torch.isfinite(y).all() and torch.equal(b(shifted(x)), y)
