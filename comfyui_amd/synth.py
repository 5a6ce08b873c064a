"""Seeded synthetic weights and activations for the HiDream MoE feed-forward at the
benchmark configurations (used by bench.py, the smoke test and the parity tests).

Everything is drawn on the CPU from one torch.Generator in state-dict order
(shared_experts.w1, w2, w3, experts.0.w1 ... experts.{E-1}.w3, gate.weight, then x),
in fp32, then cast. Shapes follow the reference model (dim 2560, 4 routed experts of
hidden 6912, top-2, shared expert of hidden 3584:
/root/reference/comfy/model_detection.py:453-470,
/root/reference/comfy/ldm/hidream/model.py:225-231,297).
"""
import math

import torch

DIM = 2560
HIDDEN_ARG = 4 * DIM          # the blocks pass hidden_dim = 4 * dim (model.py:397,473)
NUM_EXPERTS = 4
TOP_K = 2
FP8 = torch.float8_e4m3fn


def swiglu_hidden(hidden_dim, multiple_of=256):
    """Width FeedForwardSwiGLU derives from its hidden_dim argument (model.py:225-231)."""
    h = int(2 * hidden_dim / 3)
    return multiple_of * ((h + multiple_of - 1) // multiple_of)


H_ROUTED = swiglu_hidden(HIDDEN_ARG)         # 6912
H_SHARED = swiglu_hidden(HIDDEN_ARG // 2)    # 3584


def quantize_per_tensor(w_fp32):
    """scale_weight = amax/448 (fp32), W8 = (W / scale_weight) -> float8_e4m3fn."""
    s = (w_fp32.abs().amax() / 448.0).to(torch.float32)
    return (w_fp32 / s).to(FP8), s


def quantize_per_block(w_fp32):
    """One scale for each 128 x 128 block, amax/448 (fp32); W8 = (W / scale) -> float8_e4m3fn. Returns (W8, scales)."""
    n, k = w_fp32.shape
    pad = torch.nn.functional.pad(w_fp32, (0, -k % 128, 0, -n % 128))
    blocks = pad.view(pad.shape[0] // 128, 128, pad.shape[1] // 128, 128)
    s = (blocks.abs().amax((1, 3), keepdim=True).clamp_min(2.0 ** -96) / 448.0).to(torch.float32)
    return (blocks / s).view(pad.shape)[:n, :k].to(FP8).contiguous(), s[:, 0, :, 0].contiguous()


def make_weights(seed=0, dim=DIM, hidden_arg=None, num_experts=NUM_EXPERTS, sigma=0.02, generator=None, device=None):
    """fp32 master weights as a flat dict keyed like the module's state dict. `device` draws them there (its own
    generator stream: not the same numbers as on the CPU, the same distribution)."""
    hidden_arg = hidden_arg if hidden_arg is not None else 4 * dim
    g = generator if generator is not None else torch.Generator(device=device if device is not None else "cpu").manual_seed(seed)
    hs, hr = swiglu_hidden(hidden_arg // 2), swiglu_hidden(hidden_arg)
    sd = {}

    def ffn(prefix, h):
        sd[prefix + "w1.weight"] = torch.randn((h, dim), generator=g, device=device) * sigma
        sd[prefix + "w2.weight"] = torch.randn((dim, h), generator=g, device=device) * sigma
        sd[prefix + "w3.weight"] = torch.randn((h, dim), generator=g, device=device) * sigma

    ffn("shared_experts.", hs)
    for e in range(num_experts):
        ffn(f"experts.{e}.", hr)
    sd["gate.weight"] = torch.randn((num_experts, dim), generator=g, device=device) / math.sqrt(dim)
    return sd, g


def to_state_dict(master, weights="fp8", scale_input=True):
    """Cast the fp32 master weights into a loadable state dict.
    weights="bf16": all bf16. weights="fp8_block": Linear weights e4m3fn + scale_weight of each 128 x 128 block. weights="fp8": Linear weights e4m3fn + scale_weight (+ scale_input = 1.0),
    gate.weight bf16."""
    out = {}
    for k, v in master.items():
        if k == "gate.weight" or weights == "bf16":
            out[k] = v.to(torch.bfloat16)
            continue
        w8, s = quantize_per_block(v) if weights == "fp8_block" else quantize_per_tensor(v)
        out[k] = w8
        out[k.replace(".weight", ".scale_weight")] = s
        if scale_input and weights != "fp8_block":
            out[k.replace(".weight", ".scale_input")] = torch.ones((), dtype=torch.float32, device=v.device)
    return out


def make_input(generator, tokens, dim=DIM, batch=1, outlier_frac=0.0, outlier_scale=20.0):
    """x ~ N(0,1) as bf16 [batch, tokens/batch, dim]; optionally a fraction of channels scaled up."""
    x = torch.randn((tokens, dim), generator=generator)
    if outlier_frac > 0:
        n = max(1, int(round(outlier_frac * dim)))
        ch = torch.randperm(dim, generator=generator)[:n]
        x[:, ch] *= outlier_scale
    return x.to(torch.bfloat16).view(batch, tokens // batch, dim)


def make_config(name, seed=0):
    """The five benchmark configurations. Returns dict(master=..., weights="bf16"|"fp8", x=bf16 [B,S,D], name=...)."""
    master, g = make_weights(seed)
    if name == "cfg1":      # bf16 weights, 1 x 1024 tokens
        return dict(name=name, master=master, weights="bf16", x=make_input(g, 1024))
    if name == "cfg2":      # fp8 weights, 1 x 4096 tokens
        return dict(name=name, master=master, weights="fp8", x=make_input(g, 4096))
    if name == "cfg3":      # fp8 weights, 2 x 4096 tokens, 1% outlier channels x20  (headline)
        return dict(name=name, master=master, weights="fp8", x=make_input(g, 8192, batch=2, outlier_frac=0.01))
    if name.startswith("cfg5-") and name[5:].isdigit():   # cfg5-256 and cfg5-4096 are the benchmark lines
        tokens = int(name.split("-")[1])
        x = make_input(g, tokens)
        master, x = apply_routing_skew(master, x)
        return dict(name=name, master=master, weights="fp8", x=x)
    raise ValueError(name)


def apply_routing_skew(master, x, bias=(0.1875, 0.0, 0.0, -3.0), tie_every=64):
    """Routing-skew stress: the reference gate has no bias (model.py:268), so a bias is realised
    through the existing signature -- channel 0 of x is the constant 1 and Wg[e,0] = bias[e].
    Every `tie_every`-th token is zero except channel 0, so its logits are exactly the biases and
    experts 1 and 2 (equal bias) tie exactly: the lower index must win the second slot."""
    master = dict(master)
    wg = master["gate.weight"].clone()
    wg[:, 0] = torch.tensor(bias[: wg.shape[0]], dtype=wg.dtype)
    master["gate.weight"] = wg
    xf = x.float().clone()
    flat = xf.view(-1, xf.shape[-1])
    flat[:, 0] = 1.0
    flat[::tie_every, 1:] = 0.0
    return master, xf.to(torch.bfloat16)


def build_module(state_dict, weights, device, dim=DIM, hidden_arg=None, num_experts=NUM_EXPERTS,
                 fp8_matrix_mult=True, scale_input=True):
    """Instantiate comfyui_amd.hidream.MOEFeedForwardSwiGLU with the matching operations class and
    load `state_dict` into it."""
    from . import hidream, ops
    hidden_arg = hidden_arg if hidden_arg is not None else 4 * dim
    if weights == "bf16":
        operations, dtype = ops.disable_weight_init, torch.bfloat16
    elif weights == "fp8_block":
        operations, dtype = ops.block_fp8_ops, torch.bfloat16
    else:
        operations = ops.scaled_fp8_ops(fp8_matrix_mult=fp8_matrix_mult, scale_input=scale_input, override_dtype=FP8)
        dtype = torch.bfloat16
    m = hidream.MOEFeedForwardSwiGLU(dim, hidden_arg, num_experts, TOP_K, dtype=dtype, device=device,
                                     operations=operations)
    missing, unexpected = m.load_state_dict(state_dict, strict=False)
    if unexpected or [k for k in missing if not k.endswith("scale_input")]:
        raise RuntimeError(f"state dict mismatch: missing={missing} unexpected={unexpected}")
    return m.eval()
