"""fixed_k_cut of the block-scaled operators and batch_invariant of their Linears: a row's bytes whatever rows come with it."""
import ctypes

import pytest
import torch

from tests.test_gpu_block_fp8 import close, close_cast, gen, product64, segments, tokens, weight

pytestmark = pytest.mark.gpu

ROWS = (1, 2, 7, 16, 40, 130, 700, 1930, 3000, 9000)


def bytes_of(*tensors):
    return [t.contiguous().view(torch.uint8) for t in tensors]


def ways(gate_up, a_dtype, K, N):
    """(kernel, rows of a tile, K steps in LDS) for each of ROWS."""
    from comfyui_amd import _lib as L
    found = set()
    for rows in ROWS:
        a, p = L.BlockArgs(), L.BlockPlan()
        a.a_dtype, a.out_dtype, a.rows_static, a.K_static, a.N_static, a.fixed_k_cut = a_dtype, L.W_BF16, rows, K, N, 1
        L.check(L.lib.hdmoe_block_plan_get(ctypes.byref(a), gate_up, ctypes.byref(p)))
        found.add((p.kernel, p.tile_rows, p.stages))
    return found


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,N", [(2944, 4048), (528, 272)])
def test_linear(K, N, dtype):
    from comfyui_amd import _lib as L
    from comfyui_amd import functional as HF
    g = gen(K)
    x = tokens(g, max(ROWS), K, dtype)
    w, sw = weight(g, N, K)
    bias = torch.randn(N, generator=g, device="cuda").to(dtype)
    q, s = HF.quant_block_fp8(x)
    want = HF.linear_block_fp8(x, w, sw, bias=bias, fixed_k_cut=True)
    close(want[:40], *product64(q[:40], s[:40], w, sw, bias))
    for rows in ROWS:
        y = HF.linear_block_fp8(x[:rows], w, sw, bias=bias, fixed_k_cut=True)
        assert torch.equal(y, want[:rows]), rows
        qr, sr = HF.quant_block_fp8(x[:rows])
        assert torch.equal(HF.linear_block_fp8(qr, w, sw, bias=bias, scale_x=sr, out_dtype=dtype, fixed_k_cut=True), want[:rows]), rows
        # as one of many segments, read through a permutation
        perm = torch.arange(2 * rows, dtype=torch.int32, device="cuda")
        z = HF.grouped_linear_block_fp8(x[:rows], segments([0, 2 * rows - rows // 2, rows // 2]), [(w, sw, bias)] * 3, perm=perm, fixed_k_cut=True)
        assert torch.equal(z, want[:rows].repeat_interleave(2, 0)), rows
    if K > 1000:
        assert len(ways(0, L.W_BF16, K, N)) >= 3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,H", [(1040, 1552), (528, 272)])
def test_gate_up(K, H, dtype):
    from comfyui_amd import _lib as L
    from comfyui_amd import functional as HF
    g = gen(K)
    x = tokens(g, max(ROWS), K, dtype)
    ws = (*weight(g, H, K), *weight(g, H, K))
    wide = (*weight(g, 400, K), *weight(g, 400, K))
    q, s = HF.quant_block_fp8(x)
    h, sh = HF.swiglu_block_fp8(x, *ws, fixed_k_cut=True)
    h2, sh2 = HF.swiglu_block_fp8(x, *wide, fixed_k_cut=True)
    close_cast(h[:40], sh[:40], q[:40], s[:40], *ws, exact=dtype == torch.float16)
    for rows in ROWS:
        got = HF.swiglu_block_fp8(x[:rows], *ws, fixed_k_cut=True)
        assert all(map(torch.equal, bytes_of(*got), bytes_of(h[:rows], sh[:rows]))), rows
        perm = torch.arange(2 * rows, dtype=torch.int32, device="cuda")
        got = HF.grouped_swiglu_block_fp8(x[:rows], segments([rows, 0, rows]), [ws] * 3, perm=perm, shared=wide, fixed_k_cut=True)
        want = (h[:rows].view(torch.uint8).repeat_interleave(2, 0), sh[:rows].repeat_interleave(2, 0), h2[:rows], sh2[:rows])
        assert all(map(torch.equal, bytes_of(*got), bytes_of(*want))), rows
    if K > 1000 and dtype == torch.bfloat16:
        assert len(ways(1, L.W_BF16, K, H)) >= 3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_module(dtype):
    from comfyui_amd import ops, synth
    g = torch.Generator().manual_seed(2)
    l = ops.block_fp8_ops.Linear(1296, 784, bias=True, dtype=dtype, device="cuda")
    w, s = synth.quantize_per_block(torch.randn((784, 1296), generator=g))
    l.load_state_dict({"weight": w, "scale_weight": s, "bias": torch.randn(784, generator=g).to(dtype)})
    l.batch_invariant = True
    x = torch.randn((3000, 1296), generator=g).to(dtype).cuda()
    want = l(x)
    for rows in (1, 5, 30, 200):
        assert torch.equal(l(x[:rows]), want[:rows])


def test_feed_forward_and_layer():
    """Joined launches have the property if a Linear among them asks for it: the tokens of a large batch, one by one."""
    from tests.test_gpu_block_fp8_layers import layer
    m, g, synth = layer()
    f = m.experts[1]
    x = synth.make_input(g, 2000, dim=512).cuda()
    for e in (*m.experts, m.shared_experts):
        for l in (e.w1, e.w2):
            l.batch_invariant = True
    y, z = f(x), m(x)
    for rows in (1, 4, 60, 300):
        assert torch.equal(f(x[:, :rows]), y[:, :rows])
        assert torch.equal(m(x[:, :rows]), z[:, :rows])


def test_hunyuan_block():
    from comfyui_amd import hunyuan3d, ops, synth
    g = torch.Generator().manual_seed(4)
    b = hunyuan3d.MoEBlock(256, num_experts=4, ff_inner_dim=528, operations=ops.block_fp8_ops, device="cuda", dtype=torch.float16).eval()
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
    for f in (*b.experts, b.shared_experts):
        f.net[0].proj.batch_invariant = f.net[2].batch_invariant = True
    x = torch.randn((1, 2000, 256), generator=g).half().cuda()
    y = b(x)
    for rows in (1, 4, 60, 300):
        assert torch.equal(b(x[:, :rows]), y[:, :rows])
