"""Calls of the block-scaled operators that are refused before a device is looked for."""
import pytest
import torch

F8 = torch.float8_e4m3fn


def test_scales_of_16_bit_rows_are_refused_beside_a_shared_expert_too():
    """They are for e4m3fn rows: 16-bit ones would be cast anew and the scales given ignored."""
    from comfyui_amd import functional as HF
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    w, sw = torch.zeros((128, 128)).to(F8), torch.ones((1, 1))
    off = torch.tensor([0, 4], dtype=torch.int32)
    for kwargs in ({}, dict(shared=(w, sw, None), a_static=x)):
        with pytest.raises(TypeError, match="scales belong"):
            HF.grouped_linear_block_fp8(x, off, [(w, sw, None)], scale_a=torch.ones((4, 1)), **kwargs)
    with pytest.raises(ValueError, match="activations"):
        HF.grouped_linear_block_fp8(x[None], off, [(w, sw, None)], shared=(w, sw, None), a_static=x)
