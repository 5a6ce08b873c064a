"""set_weight and convert_weight of block-scaled Linears on the device, where a block's scale is zero."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("delta", [0.0, 3.0])
def test_a_block_without_a_scale_stays_zero(dtype, delta):
    from comfyui_amd import ops
    l = ops.block_fp8_ops.Linear(272, 144, bias=False, device="cuda")
    scales = torch.tensor([[0.5, 0.0, 2.0], [0.25, 1.0, 0.0]], device="cuda")
    with torch.no_grad():
        l.scale_weight.copy_(scales)
    codes = (torch.randn((144, 272), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * 50).to(torch.float8_e4m3fn).float()
    codes[:128, 128:256] = 0
    codes[128:, 256:] = 0
    full = l.convert_weight(codes.to(dtype))
    assert full.dtype == dtype
    full[:128, 128:256] += delta
    full[128:, 256:] += delta
    l.set_weight(full, inplace_update=True, seed=1)
    again = l.weight.float()
    assert (again[:128, 128:256] == 0).all() and (again[128:, 256:] == 0).all()
    # the other scales are powers of two: exact values, which the device's rounding leaves as they are but for 2^-9 of them at most
    assert (again != codes).float().mean() < 2.0 ** -8
    x = torch.randn((5, 272), device="cuda").bfloat16()
    y = l(x)
    assert torch.isfinite(y).all()
