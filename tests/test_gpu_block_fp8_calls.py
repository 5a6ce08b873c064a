"""Who makes the modules' calls of the block-scaled operators: the compiled functions, wherever the tensors are as they take them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class Watched:
    """The compiled functions, and what became of each call."""

    def __init__(self, module):
        self.module, self.calls = module, []

    def __getattr__(self, name):
        f = getattr(self.module, name)

        def call(*args):
            r = f(*args)
            self.calls.append((name, r is not None))
            return r

        return call


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [3, 200])
def test_hunyuan_block(tokens, dtype, monkeypatch):
    from comfyui_amd import functional as HF
    from comfyui_amd import hunyuan3d, ops, synth
    g = torch.Generator().manual_seed(tokens)
    b = hunyuan3d.MoEBlock(256, num_experts=4, ff_inner_dim=528, operations=ops.block_fp8_ops, device="cuda", dtype=dtype).eval()
    with torch.no_grad():
        for name, p in b.state_dict().items():
            if name.endswith("scale_weight"):
                continue
            v = torch.randn(p.shape, generator=g) * (0.05 if p.dim() == 2 else 0.5)
            if p.dtype == torch.float8_e4m3fn:
                q, s = synth.quantize_per_block(v)
                p.copy_(q)
                b.state_dict()[name.replace("weight", "scale_weight")].copy_(s)
            else:
                p.copy_(v)
    x = torch.randn((1, tokens, 256), generator=g).to(dtype).cuda()
    want = b(x)
    watched = Watched(HF._block_calls)
    monkeypatch.setattr(HF, "_block_calls", watched)
    assert torch.equal(b(x), want)
    assert [c for c in watched.calls if c[0] == "grouped_linear"] == [("grouped_linear", True)] * 2
    assert all(ok for _, ok in watched.calls)
