"""The operations class of weights with a scale for each block of 128, its hooks, checkpoints with such weights: no device."""
import torch
from safetensors.torch import save_file

from comfyui_amd import checkpoint as C
from comfyui_amd import ops, synth

FP8 = torch.float8_e4m3fn


def test_parameters_and_hooks():
    l = ops.block_fp8_ops.Linear(272, 144, bias=True, dtype=torch.float16)
    assert l.weight.dtype == FP8 and l.scale_weight.dtype == torch.float32 and tuple(l.scale_weight.shape) == (2, 3)
    assert l.bias.dtype == torch.float16 and not l.scale_weight.requires_grad
    assert sorted(l.state_dict()) == ["bias", "scale_weight", "weight"]
    assert l.comfy_cast_weights and l.weight_function == [] and l.bias_function == []
    assert ops.block_fp8_ops.Linear(16, 16, bias=False).bias is None
    assert ops.pick_operations(FP8, torch.bfloat16, block_scales=True) is ops.block_fp8_ops


def test_convert_and_set_weight():
    g = torch.Generator().manual_seed(1)
    l = ops.block_fp8_ops.Linear(272, 144, bias=False)
    with torch.no_grad():
        l.scale_weight.copy_(torch.rand((2, 3), generator=g) + 0.5)
    w = (torch.randn((144, 272), generator=g) * 50).to(FP8)
    l.weight = torch.nn.Parameter(w, requires_grad=False)
    full = l.convert_weight(w.float())
    want = w.float().clone()
    for i in range(2):
        for j in range(3):
            want[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128] *= l.scale_weight[i, j]
    assert torch.equal(full, want)
    again = l.set_weight(full, return_weight=True, seed=7)
    # The stored bytes come back but for the host's random digit: it is an fp16 u in [0, 1) added to a mantissa in eighths m < 8 in fp16, whose
    # step is 2^-8 there or finer, so an m that is whole is taken for the next one if u >= 1 - 2^-9: 2^-9 of the values at most, 77 of these
    # 39168 with a deviation of 9; 2^-8 is 8 of those away. (v * s) / s itself is v but for 2^-23, less than fp16 holds.
    assert again.dtype == FP8 and (again.float() != w.float()).float().mean() < 2.0 ** -8
    mine = w.float().clone()
    assert l.convert_weight(mine, inplace=True) is mine and torch.equal(mine, want)
    l.set_weight(torch.zeros_like(full), seed=1)
    assert l.weight.dtype == FP8 and (l.weight.float() == 0).all()


def test_quantize_per_block():
    g = torch.Generator().manual_seed(2)
    w = torch.randn((200, 300), generator=g)
    w[:128, 128:256] *= 100
    w[128:, 256:] = 0
    q, s = synth.quantize_per_block(w)
    assert tuple(s.shape) == (2, 3) and q.shape == w.shape
    for i in range(2):
        for j in range(3):
            b = w[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128]
            v = q[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].float()
            assert s[i, j] == b.abs().max().clamp_min(2.0 ** -96) / 448
            # half an e4m3fn step: 2^-4 of the value, or 2^-10 of the scale below the normal range
            assert ((v * s[i, j] - b).abs() <= b.abs() * 2.0 ** -4 * (1 + 2.0 ** -10) + s[i, j] * 2.0 ** -10).all()


def test_checkpoint_with_block_scales(tmp_path):
    master, _ = synth.make_weights(3, dim=256, hidden_arg=1024, num_experts=3)
    sd = {f"model.blocks.0.ff_i.{k}": v for k, v in synth.to_state_dict(master, "fp8_block").items()}
    sd["model.scaled_fp8"] = C.scaled_fp8_marker(FP8, True)
    path = str(tmp_path / "m.safetensors")
    save_file(sd, path)
    for source in (path, dict(sd)):
        modules, info = C.load_moe_layers(source, prefix="model.")
        assert info["operations"] is ops.block_fp8_ops
        (m,) = modules.values()
        for k, v in m.state_dict().items():
            want = sd[f"model.blocks.0.ff_i.{k}"]
            assert v.dtype == want.dtype and torch.equal(v.float(), want.float()), k
    # one scale a tensor: as before
    sd = {f"b.{k}": v for k, v in synth.to_state_dict(master, "fp8").items()}
    sd["scaled_fp8"] = C.scaled_fp8_marker(FP8, True)
    assert C.load_moe_layers(sd)[1]["operations"] is not ops.block_fp8_ops
