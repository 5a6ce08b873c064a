"""Layer norm of rows whose values have much in common: the first mean of a row is off by up to 84 * 2^-24 of the values (norm64), which eps in the
root magnifies where the rest is small. What is left of it after the second sum is that much of the differences alone."""
import pytest
import torch

from tests import norm64
from tests.norm64 import U, close
from tests.test_gpu_norm import check, gains, gen

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def tight(x, eps):
    """norm64.stats for a mean that is corrected by that of the differences from it. `first`: how far off it is before. The variance is the sum of squares of
    differences that have this in them too, less its square: 84 * 2^-24 of that beside what norm64 has. Two roundings of the differences themselves."""
    x = x.double()
    c = x - x.mean(-1, keepdim=True)
    r = (c.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    n = c * r
    first = 84 * U * x.abs().mean(-1, keepdim=True)
    dm = 84 * U * (c.abs().mean(-1, keepdim=True) + first)
    return n, r, dm * r + (50 * U + (dm * r).pow(2) + 84 * U * (first * r).pow(2)) * n.abs() + 2 * U * (c.abs() + first) * r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 2100])
@pytest.mark.parametrize("D,value", [(1000, 29952.0), (1000, 1000.0), (4095, 240.0), (6912, 29952.0), (6912, 0.1), (333, -7.3), (2560, 3.0), (16383, 511.0)])
def test_equal_values(dtype, rows, D, value):
    """Differences of 0: the result is the bias to the bit, the weight's gradient 0, dx = r (g - mean(g)) with the variance's rounding (see tight) in r."""
    from comfyui_amd import functional as HF
    g = gen(D)
    eps = 1e-5
    x = torch.full((rows, D), value, device="cuda", dtype=dtype)
    w, b = gains(g, D, dtype)
    dy = torch.randn((rows, D), generator=g, device="cuda").to(dtype)
    assert torch.equal(HF.layer_norm(x, w, b, eps=eps), b.expand(rows, D))
    assert not HF.layer_norm(x, eps=eps).any()
    dx, dw, db = HF.layer_norm_backward(dy, x, w, b, eps=eps)
    assert not dw.any()
    (e, ee), _, (eb, eeb) = norm64.backward(dy, x, w.double(), eps)
    gd = (dy.double() * w.double()).abs()
    room = eps ** -0.5 * (4 * U * gd + 84 * U * gd.mean(-1, keepdim=True)) + e.abs() * (50 * U + 42 * U * (84 * U * abs(float(x[0, 0]))) ** 2 / eps)
    close(dx, e, room, "dx")
    close(db, eb, eeb, "db")


@pytest.mark.parametrize("rows,D", [(1, 1000), (77, 4095), (2500, 1000), (2100, 2200), (40, 6912), (5, 16383), (3, 333)])
@pytest.mark.parametrize("offset,size", [(1e4, 1.0), (-300.0, 0.01), (0.0, 1.0)])
def test_large_offsets(rows, D, offset, size, monkeypatch):
    monkeypatch.setattr(norm64, "stats", tight)
    g = gen(rows + D)
    x = torch.randn((rows, D), generator=g, device="cuda") * size + offset
    check(x, *gains(g, D, torch.float32), torch.randn((rows, D), generator=g, device="cuda"), 1e-5)
    check(x, None, None, torch.randn((rows, D), generator=g, device="cuda"), 0.0)


def test_modulated_gradients_with_an_offset(monkeypatch):
    from comfyui_amd import functional as HF
    monkeypatch.setattr(norm64, "stats", tight)
    g = gen(9)
    B, L, D = 3, 700, 1000
    x = torch.randn((B * L, D), generator=g, device="cuda") + 1e4
    dy = torch.randn(x.shape, generator=g, device="cuda")
    scale = 0.4 * torch.randn((B, D), generator=g, device="cuda")
    dx, ds, dsh = HF.ln_modulate_backward(dy, x, scale, L, eps=1e-6)
    (e, ee), (es, ees), (eb, eeb) = norm64.backward(dy.view(B, L, D), x.view(B, L, D), 1 + scale.double()[:, None], 1e-6, rows_dim=1)
    close(dx.view(B, L, D), e, ee, "dx")
    close(ds, es, ees, "dscale")
    close(dsh, eb, eeb, "dshift")


def test_rows_past_the_squares_range():
    """fp32 rows whose squares are past the largest number: an infinite variance, so 0, as torch's has it; equal ones among them are equal all the same."""
    from comfyui_amd import functional as HF
    x = torch.ones((3, 700), device="cuda") * 1e25
    x[1, ::2] = -1e25
    x[2, ::3] = 3e25
    y = HF.layer_norm(x)
    assert not y.any()
