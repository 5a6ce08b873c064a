"""convert_weight and set_weight of Linears with a scale for each block of 128, where a block's scale is zero or next to it: no device."""
import pytest
import torch

from comfyui_amd import ops

FP8 = torch.float8_e4m3fn


def linear(scales):
    l = ops.block_fp8_ops.Linear(272, 144, bias=False)
    with torch.no_grad():
        l.scale_weight.copy_(torch.tensor(scales))
    g = torch.Generator().manual_seed(3)
    w = (torch.randn((144, 272), generator=g) * 50).to(FP8)
    l.weight = torch.nn.Parameter(w, requires_grad=False)
    return l


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("delta", [0.0, 3.0])
def test_a_block_without_a_scale_stays_zero(dtype, delta):
    """An all-zero block stored with the plain amax / 448: its codes stay zeros through a patch, they do not become 0 / 0."""
    l = linear([[0.5, 0.0, 2.0], [0.25, 1.0, 0.0]])
    codes = l.weight.float()
    codes[:128, 128:256] = 0
    codes[128:, 256:] = 0
    full = l.convert_weight(codes.to(dtype))
    assert full.dtype == dtype
    full[:128, 128:256] += delta
    full[128:, 256:] += delta
    again = l.set_weight(full, return_weight=True, seed=1).float()
    assert torch.isfinite(again).all()
    assert (again[:128, 128:256] == 0).all() and (again[128:, 256:] == 0).all()
    # the other blocks' scales are powers of two: codes come back but for the host's random digit, 2^-9 of them
    assert (again != codes).float().mean() < 2.0 ** -8
    inplace = codes.to(dtype)
    assert l.convert_weight(inplace, inplace=True) is inplace


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scales_below_what_the_weights_type_holds(dtype):
    """2^-96 / 448 (a block of zeros as synth.quantize_per_block stores it) is zero in fp16, and 2^-26 is not what fp16 makes of it."""
    l = linear([[1.0, 2.0 ** -96 / 448, 2.0 ** -26], [1.0, 1.0, 1.0]])
    codes = l.weight.float()
    codes[:128, 128:256] = 0
    again = l.set_weight(l.convert_weight(codes.to(dtype)), return_weight=True, seed=2).float()
    assert torch.isfinite(again).all() and (again[:128, 128:256] == 0).all()
    # products with 2^-26 are subnormal in fp16, whole multiples of 2^-24: off by half of that at most, two of the codes' units; the next code above
    # or below is 2^-3 of the value away, or 2^-9
    if dtype == torch.float16:
        limit = 2 + (codes[:128, 256:].abs() + 2) * 2.0 ** -3
        assert ((again - codes)[:128, 256:].abs() <= limit).all()
    else:
        assert (again != codes).float().mean() < 2.0 ** -8
