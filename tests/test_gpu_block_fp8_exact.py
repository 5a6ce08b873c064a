"""Gate/up with exact products: up to 64 rows in every type, with fp16 activations and with exact=True at any size.

The operands make the difference plain. In every block of 128 two products of 2^16 cancel, each among seven of 2^2, which an e4m3fn matrix instruction that
cuts at 2^-13 of the largest of eight neighbours loses: 56 of a block's sum of 500, and with it a fifth of silu(g) * u. All sums are whole numbers
below 2^24, so that exact products give g and u to the bit in any order; the fp32 exponential, quotient and products of silu(g) * u add a few 2^-23, the
scale's quotient one: 2^-20 in all."""
import pytest
import torch

from tests.test_gpu_block_fp8 import F8, close_cast, gen, product64, segments, silu64, tokens, weight

pytestmark = pytest.mark.gpu


def operands(rows, K, N):
    x = torch.full((rows, K), 2.0, device="cuda")
    w = torch.full((N, K), 2.0, device="cuda")
    x[:, 0::128], x[:, 8::128], x[:, 16::128] = 256, -256, 448      # 448: the cast's scale is 1
    w[:, 0::128], w[:, 8::128], w[:, 16::128] = 256, 256, 0
    return x, (w.to(F8), torch.full((-(-N // 128), -(-K // 128)), 2.0 ** -12, device="cuda"))


def is_exact(h, sh, K):
    g = torch.tensor(K // 128 * 500 * 2.0 ** -12, dtype=torch.float64, device="cuda")
    want = silu64(g) * g
    value = h.double() * sh.double().repeat_interleave(128, 1)[:, :h.shape[1]]
    return ((value / want - 1).abs() <= 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, F8])
@pytest.mark.parametrize("T", [1, 4, 8, 21, 32])
def test_a_layer_of_few_tokens(T, dtype):
    """2 T routed rows, T of the shared expert: the sizes of the package's own layer."""
    from comfyui_amd import functional as HF
    x, w = operands(T, 2560, 6912)
    _, shared = operands(1, 2560, 3584)
    scale = torch.ones((20, T), device="cuda").t() if dtype == F8 else None
    perm = torch.arange(2 * T, dtype=torch.int32, device="cuda")
    for sizes in ([2 * T, 0, 0, 0], [T, 0, T - T // 2, T // 2]):
        got = HF.grouped_swiglu_block_fp8(x.to(dtype), segments(sizes), [(*w, *w)] * 4, scale_a=scale, perm=perm, shared=(*shared, *shared))
        assert is_exact(*got[:2], 2560) and is_exact(*got[2:], 2560)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, F8])
@pytest.mark.parametrize("rows,E,K,N", [(64, 0, 2560, 6912), (64, 4, 2560, 6912), (9, 4, 2560, 6912), (63, 8, 640, 4112), (64, 32, 256, 272), (2, 0, 16384, 272)])
def test_up_to_64_rows(rows, E, K, N, dtype):
    from comfyui_amd import functional as HF
    x, w = operands(rows, K, N)
    x, scale = x.to(dtype), torch.ones((K // 128, rows), device="cuda").t() if dtype == F8 else None
    if E == 0:
        got = HF.swiglu_block_fp8(x, *w, *w, scale_x=scale)
    else:
        got = HF.grouped_swiglu_block_fp8(x, segments([rows - (E - 2) * (rows // E), 0] + [rows // E] * (E - 2)), [(*w, *w)] * E, scale_a=scale)
    assert is_exact(*got, K)


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, F8])
@pytest.mark.parametrize("rows", [5, 65, 700, 5000])
def test_when_asked(rows, dtype, fixed):
    """exact=True, alone and with fixed_k_cut; on random operands as well."""
    from comfyui_amd import functional as HF
    K, N = 1280, 1552
    x, w = operands(rows, K, N)
    x, scale = x.to(dtype), torch.ones((K // 128, rows), device="cuda").t() if dtype == F8 else None
    assert is_exact(*HF.swiglu_block_fp8(x, *w, *w, scale_x=scale, exact=True, fixed_k_cut=fixed), K)
    off = segments([rows // 2, 0, rows - rows // 2])
    assert is_exact(*HF.grouped_swiglu_block_fp8(x, off, [(*w, *w)] * 3, scale_a=scale, exact=True, fixed_k_cut=fixed), K)
    if dtype != F8:
        g = gen(rows)
        x, ws = tokens(g, rows, K, dtype), (*weight(g, N, K), *weight(g, N, K))
        q, s = HF.quant_block_fp8(x)
        h, sh = HF.swiglu_block_fp8(x, *ws, exact=True, fixed_k_cut=fixed)
        close_cast(h, sh, q, s, *ws, exact=True)


@pytest.mark.parametrize("rows", [1, 30, 400])
def test_both_ways_to_make_the_call(rows, monkeypatch):
    from comfyui_amd import functional as HF
    g = gen(rows)
    x, up = tokens(g, rows, 656), (*weight(g, 272, 656), *weight(g, 272, 656))
    w = weight(g, 272, 656)
    calls = [lambda: HF.swiglu_block_fp8(x, *up, exact=True), lambda: HF.swiglu_block_fp8(x, *up, fixed_k_cut=True),
             lambda: HF.grouped_swiglu_block_fp8(x, segments([rows, 0]), [up] * 2, exact=True, fixed_k_cut=True, shared=up),
             lambda: HF.linear_block_fp8(x, *w, fixed_k_cut=True), lambda: HF.grouped_linear_block_fp8(x, segments([rows]), [(*w, None)], fixed_k_cut=True)]
    made = [f() for f in calls]
    monkeypatch.setattr(HF, "_stream_here", lambda t: None)
    for a, f in zip(made, calls):
        b = f()
        for t, u in zip(*((v if isinstance(v, tuple) else (v,)) for v in (a, b))):
            assert torch.equal(t.contiguous().view(torch.uint8), u.contiguous().view(torch.uint8))


def test_product64_agrees_with_the_pattern():
    """The oracle's own view of these operands."""
    x, w = operands(3, 640, 128)
    y, _ = product64(x.to(F8), torch.ones((3, 5), device="cuda"), *w, exact=True)
    assert (y == 5 * 500 * 2.0 ** -12).all()
