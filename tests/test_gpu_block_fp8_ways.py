"""Ways to run the block-scaled contractions that the other lists of sizes leave out: K of a single block on the tile kernels, tiles that end in a single
row, 256-row tiles of two parts on one segment. Tolerances are those of test_gpu_block_fp8."""
import pytest
import torch

from tests.test_gpu_block_fp8 import close, close_cast, gen, product64, segments, tokens, weight

pytestmark = pytest.mark.gpu

# (rows of each segment, as segments of experts or one dense call, K, N)
LINEAR = [([1930], False, 2944, 4048), ([129], False, 16, 5536), ([257], False, 112, 4096), ([3000], False, 128, 2048), ([385, 0, 1, 64], True, 96, 4176),
          ([129, 1, 300], True, 128, 5536), ([1, 1, 129, 257], True, 16, 6000)]
GATE_UP = [([100], False, 112, 128), ([129], False, 16, 640), ([8321], False, 96, 144), ([16449], False, 48, 144), ([20225], False, 128, 2048),
           ([526], False, 128, 6544), ([65], False, 128, 6544), ([8065, 1, 100, 0], True, 80, 144), ([12000, 4100, 200, 1], True, 112, 144),
           ([12000, 4100, 200, 1], True, 16, 144), ([257, 1, 0, 65], True, 32, 8176), ([65, 1, 0, 66], True, 128, 8176), ([20000, 225, 1], True, 112, 2048),
           ([100, 1, 29], True, 80, 128)]


@pytest.mark.parametrize("sizes,many,K,N", LINEAR)
def test_linear(sizes, many, K, N):
    from comfyui_amd import functional as HF
    rows = sum(sizes)
    g = gen(rows + K + N)
    x = tokens(g, rows, K)
    q, s = HF.quant_block_fp8(x)
    experts = [(*weight(g, N, K), None) for _ in sizes]
    off = segments(sizes)
    b = off.tolist()
    for a, scale in ((x, None), (q, s)):
        y = HF.grouped_linear_block_fp8(a, off, experts, scale_a=scale) if many else HF.linear_block_fp8(a, *experts[0][:2], scale_x=scale)
        for (w, sw, _), lo, hi in zip(experts, b, b[1:]):
            if hi > lo:
                close(y[lo:hi], *product64(q[lo:hi], s[lo:hi], w, sw))


@pytest.mark.parametrize("sizes,many,K,N", GATE_UP)
def test_gate_up(sizes, many, K, N):
    from comfyui_amd import functional as HF
    rows = sum(sizes)
    g = gen(rows + K + N)
    x = tokens(g, rows, K)
    q, s = HF.quant_block_fp8(x)
    experts = [(*weight(g, N, K), *weight(g, N, K)) for _ in sizes]
    off = segments(sizes)
    b = off.tolist()
    for a, scale in ((x, None), (q, s)):
        h, sh = HF.grouped_swiglu_block_fp8(a, off, experts, scale_a=scale) if many else HF.swiglu_block_fp8(a, *experts[0], scale_x=scale)
        for ws, lo, hi in zip(experts, b, b[1:]):
            if hi > lo:
                close_cast(h[lo:hi], sh[lo:hi], q[lo:hi], s[lo:hi], *ws)
