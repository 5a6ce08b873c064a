"""Layer norm without a device: the 64-bit formulas that the device tests compare with, against autograd and against differences, and the
calls that are refused before a device is looked for."""
import ctypes

import pytest
import torch

from tests import norm64


def test_formulas_against_autograd_and_differences():
    g = torch.Generator().manual_seed(1)
    x = torch.randn((7, 33), generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(33, generator=g, dtype=torch.float64, requires_grad=True)
    b = torch.randn(33, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn((7, 33), generator=g, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(x, (33,), w, b, 1e-5)
    want = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        assert torch.allclose(norm64.norm(x, w, b, 1e-5)[0], y, rtol=1e-12, atol=1e-12)
        (dx, _), (dw, _), (db, _) = norm64.backward(dy, x, w, 1e-5)
        for a, c in zip((dx, dw, db), want):
            assert torch.allclose(a, c, rtol=1e-10, atol=1e-10)
        v = torch.randn(x.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        along = lambda s: (norm64.norm(x + s * h * v, w, b, 1e-5)[0] * dy).sum()  # noqa: E731
        assert abs((along(1) - along(-1)) / (2 * h) - (dx * v).sum()) < 1e-6 * dx.abs().sum()


def test_refusals():
    from comfyui_amd import functional as HF
    x = torch.zeros((4, 16), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        HF.layer_norm(x.to(torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        HF.layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        HF.layer_norm_backward(x, x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        HF.ln_modulate_backward(x, x, x[:1], 4)


def test_library_refusals_without_a_device():
    from comfyui_amd import _lib
    L = _lib.lib
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    assert L.hdmoe_layer_norm(1, p, 4, 16, 0, None, None, 1e-5, p, None) == _lib.E_SHAPE       # no such type
    assert L.hdmoe_layer_norm(_lib.T_BF16, p, 4, 16, _lib.T_F16, p, None, 1e-5, p, None) == _lib.E_SHAPE
    assert L.hdmoe_layer_norm(_lib.T_BF16, p, 4, 0, 0, None, None, 1e-5, p, None) == _lib.E_SHAPE
    assert L.hdmoe_layer_norm(_lib.T_BF16, p, 4, 16385, 0, None, None, 1e-5, p, None) == _lib.E_SHAPE
    assert L.hdmoe_layer_norm(_lib.T_BF16, p, 4, 16, 0, None, None, -1.0, p, None) == _lib.E_SHAPE
    assert L.hdmoe_layer_norm(_lib.T_BF16, p, 4, 16, 0, None, None, float("nan"), p, None) == _lib.E_SHAPE
    assert L.hdmoe_layer_norm(_lib.T_BF16, None, 4, 16, 0, None, None, 1e-5, p, None) == _lib.E_NULL
    assert L.hdmoe_layer_norm(_lib.T_BF16, None, 0, 16, 0, None, None, 1e-5, None, None) == 0   # nothing to do

    def backward(**kwargs):
        a = _lib.NormGradArgs()
        a.dtype, a.gain_dtype, a.D, a.rows, a.rows_per_group, a.eps = _lib.T_BF16, _lib.T_F32, 64, 1000, 1000, 1e-5
        a.dy = a.x = a.weight = a.dx = a.dweight = a.dbias = p
        for k, v in kwargs.items():
            setattr(a, k, v)
        return L.hdmoe_layer_norm_backward(ctypes.byref(a), None)

    need = L.hdmoe_layer_norm_backward_workspace_bytes(1000, 64, 1000)
    assert need > 0
    assert backward(dtype=3) == _lib.E_SHAPE
    assert backward(gain_dtype=_lib.T_F16) == _lib.E_SHAPE
    assert backward(D=16385) == _lib.E_SHAPE
    assert backward(rows_per_group=300) == _lib.E_SHAPE
    assert backward(rows_per_group=0) == _lib.E_SHAPE
    assert backward(rows=-1) == _lib.E_SHAPE
    assert backward(rows=1 << 23, rows_per_group=1) == _lib.E_SHAPE        # more threads than a launch has
    assert backward(eps=-1.0) == _lib.E_SHAPE
    assert backward(dy=None) == _lib.E_NULL
    assert backward() == _lib.E_WORKSPACE
    assert backward(workspace=p, workspace_bytes=need - 1) == _lib.E_WORKSPACE
    assert backward(workspace=p + 4, workspace_bytes=need) == _lib.E_WORKSPACE
    assert L.hdmoe_layer_norm_backward(None, None) == _lib.E_NULL
    assert L.hdmoe_layer_norm_backward_workspace_bytes(3, 64, 3) == 0      # one block: its sums are the result
    assert L.hdmoe_layer_norm_backward_workspace_bytes(10, 64, 3) == 0     # refused by the call
