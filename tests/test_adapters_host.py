"""Adapters of many requests without a device: the 64-bit formulas against autograd and differences, refusals, structures and workspace sizes."""
import ctypes
import os
import subprocess

import pytest
import torch

from tests import adapters64

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_formulas_against_autograd_and_differences():
    g = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    x, base, a, b = rand(12, 9), rand(12, 7), rand(3, 2, 9), rand(3, 7, 2)
    scale, index = rand(3).abs(), torch.tensor([2, -1, 0, 2], dtype=torch.int32)

    def f(x, a, b):
        out = []
        for t in range(12):
            i = int(index[t // 3])
            out.append(base[t] if i < 0 else base[t] + scale[i] * (b[i] @ (a[i] @ x[t])))
        return torch.stack(out)

    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    y = f(*leaves)
    dy = rand(12, 7)
    want = torch.autograd.grad(y, leaves, dy)
    assert torch.allclose(adapters64.forward(base, x, a, b, scale, index)[0], y.detach(), rtol=1e-12, atol=1e-12)
    got = adapters64.backward(dy, x, a, b, scale, index)
    for (v, _), w in zip(got, want):
        assert torch.allclose(v, w, rtol=1e-12, atol=1e-12)
    h, moves = 1e-6, [rand(*t.shape) for t in (x, a, b)]
    along = lambda s: (f(*(t + s * h * m for t, m in zip((x, a, b), moves))) * dy).sum()  # noqa: E731
    told = sum((v * m).sum() for (v, _), m in zip(got, moves))
    assert abs((along(1) - along(-1)) / (2 * h) - told) < 1e-6 * (1 + abs(told))


def test_refusals():
    from comfyui_amd import functional as HF
    x = torch.zeros((4, 16), dtype=torch.bfloat16)
    a, b = torch.zeros((2, 8, 16), dtype=torch.bfloat16), torch.zeros((2, 24, 8), dtype=torch.bfloat16)
    scale, index = torch.ones(2), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        HF.add_adapters(x.float(), x.float(), a, b, scale, index)
    with pytest.raises(RuntimeError, match="no CPU path"):
        HF.add_adapters(x, x, a, b, scale, index)
    with pytest.raises(RuntimeError, match="no CPU path"):
        HF.add_adapters_backward(x, x, a, b, scale, index)


def _args(**kwargs):
    from comfyui_amd import _lib
    buf = (ctypes.c_char * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    a = _lib.AdapterArgs()
    a.dtype, a.rows, a.requests, a.K, a.N, a.n, a.R = _lib.T_BF16, 64, 4, 4096, 65536, 2, 16
    for name in ("x", "a", "b", "scale", "index", "base", "out", "dy", "dx", "da", "db"):
        setattr(a, name, p)
    for k, v in kwargs.items():
        setattr(a, k, v)
    a.keep = buf
    return a


def test_library_refusals_without_a_device():
    from comfyui_amd import _lib
    L = _lib.lib
    for fn in (L.hdmoe_add_adapters, L.hdmoe_add_adapters_backward):
        assert fn(None, None) == _lib.E_NULL
        for bad in (dict(dtype=_lib.T_F32), dict(dtype=1), dict(rows=-1), dict(requests=0), dict(requests=3), dict(requests=-4), dict(K=0), dict(N=0), dict(n=0),
                    dict(n=4097), dict(R=0), dict(R=257), dict(K=1 << 25), dict(rows=1 << 30, requests=1, N=1 << 24)):
            assert fn(ctypes.byref(_args(**bad)), None) == _lib.E_SHAPE, bad
        for missing in ("x", "a", "b", "scale", "index"):
            assert fn(ctypes.byref(_args(**{missing: None})), None) == _lib.E_NULL, missing
        assert fn(ctypes.byref(_args()), None) == _lib.E_WORKSPACE
        assert b"workspace" in L.hdmoe_last_error()
    assert L.hdmoe_add_adapters(ctypes.byref(_args(base=None)), None) == _lib.E_NULL
    assert L.hdmoe_add_adapters_backward(ctypes.byref(_args(dx=None)), None) == _lib.E_NULL
    assert L.hdmoe_add_adapters_backward(ctypes.byref(_args(db=None)), None) == _lib.E_NULL
    assert L.hdmoe_add_adapters(ctypes.byref(_args(rows=0, requests=0)), None) == 0
    need = L.hdmoe_adapters_workspace_bytes(ctypes.byref(_args()), 1)
    assert need > L.hdmoe_adapters_workspace_bytes(ctypes.byref(_args()), 0) > 0
    a = _args()
    a.workspace, a.workspace_bytes = a.x, need - 1
    assert L.hdmoe_add_adapters_backward(ctypes.byref(a), None) == _lib.E_WORKSPACE
    a.workspace, a.workspace_bytes = a.x + 4, need
    assert L.hdmoe_add_adapters_backward(ctypes.byref(a), None) == _lib.E_WORKSPACE
    assert L.hdmoe_adapters_workspace_bytes(ctypes.byref(_args(R=300)), 0) == 0


@pytest.mark.parametrize("backward", [0, 1])
def test_workspace_stays_within_reason(backward):
    """Narrow values (a few copies of [rows, R]; none where one launch does it all) and, backward, a few copies of the gradients."""
    from comfyui_amd import _lib
    for rows, requests, K, N, n, R in ((1, 1, 2560, 6912, 4, 16), (48, 48, 6912, 2560, 40, 32), (16384, 4, 2560, 6912, 2, 64), (999, 3, 2048, 8192, 2, 24),
                                       (100000, 100000, 640, 640, 7, 256), (8192, 2, 2560, 6912, 1, 8)):
        nb = _lib.lib.hdmoe_adapters_workspace_bytes(ctypes.byref(_args(rows=rows, requests=requests, K=K, N=N, n=n, R=R)), backward)
        assert (0 if rows == 1 and not backward else 1) <= nb <= 2 * 16 * (rows * R * 4 + 256) + (64 * n * R * (K + N) * 4 if backward and n < 4 else 2 * 4 * n * R * (K + N) * 4) + 1024


def test_parts_of_many_adapters_stay_bounded():
    """Parts of the gradients hold every adapter: with thousands of them the rows are not cut into as many runs."""
    from comfyui_amd import _lib
    for rows, requests, n, R in ((16384, 4, 4096, 64), (65536, 8, 1024, 128), (512, 4, 4096, 256), (8192, 8192, 30, 32)):
        nb = _lib.lib.hdmoe_adapters_workspace_bytes(ctypes.byref(_args(rows=rows, requests=requests, K=2560, N=6912, n=n, R=R)), 1)
        assert 0 < nb <= (1 << 30) + 2 * 16 * (rows * R * 4 + 256) + 160 * n * 4 + 4096, (rows, n, R, nb)


def test_launches_that_are_too_large_are_refused():
    from comfyui_amd import _lib
    L = _lib.lib
    for fn in (L.hdmoe_add_adapters, L.hdmoe_add_adapters_backward):
        for bad in (dict(rows=1 << 23, requests=1 << 23, K=16, N=16, n=64), dict(rows=1 << 22, requests=1 << 21, K=16, N=16384, n=64),
                    dict(rows=1 << 28, requests=1, K=16, N=16, R=256), dict(rows=1 << 30, requests=1, K=16, N=16)):
            assert fn(ctypes.byref(_args(**bad)), None) == _lib.E_SHAPE, bad
            assert L.hdmoe_adapters_workspace_bytes(ctypes.byref(_args(**bad)), 1) == 0
        for good in (dict(rows=1 << 20, requests=1 << 20, K=2560, N=2560, n=64), dict(rows=1 << 24, requests=4, K=64, N=64, R=256)):
            assert fn(ctypes.byref(_args(**good)), None) == _lib.E_WORKSPACE, good
    assert L.hdmoe_add_adapters_backward(ctypes.byref(_args(n=4096, R=256, K=4096, N=4096)), None) == _lib.E_SHAPE


def test_results_over_inputs_are_refused():
    """base itself takes the result; x, an adapter or a part of base does not, x that is base neither."""
    from comfyui_amd import _lib
    L = _lib.lib
    sizes = dict(rows=64, requests=64, K=256, N=256, n=2, R=16)
    buf = (ctypes.c_char * (1 << 20))()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    at = {name: p + i * (1 << 16) for i, name in enumerate(("x", "a", "b", "base", "workspace"))}      # 32 KB each at most, but for the workspace
    for name, shift in (("x", 0), ("x", 32766), ("a", 2), ("b", -32766), ("base", 2), ("base", -2)):
        args = _args(**sizes, **at, out=at[name] + shift, workspace_bytes=1 << 19)
        assert L.hdmoe_add_adapters(ctypes.byref(args), None) == _lib.E_SHAPE and b"overlaps" in L.hdmoe_last_error(), (name, shift)
    args = _args(**sizes, **{**at, "base": at["x"]}, out=at["x"], workspace_bytes=1 << 19)
    assert L.hdmoe_add_adapters(ctypes.byref(args), None) == _lib.E_SHAPE


def test_struct_layouts_match_what_a_c_compiler_sees(tmp_path):
    from comfyui_amd import _lib
    structs = {"hdmoe_norm_grad_args": _lib.NormGradArgs, "hdmoe_adapter_args": _lib.AdapterArgs}
    lines = []
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hdmoe.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = dict(l.split() for l in subprocess.check_output([str(exe)], text=True).splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"


def test_sizes_that_a_c_int_does_not_hold(monkeypatch):
    from comfyui_amd import functional as HF
    monkeypatch.setattr(HF, "_need_hip", lambda *a: None)
    make = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    scale, index = make(2, dtype=torch.float32), make(4, dtype=torch.int32)
    for rows, N in (((1 << 32) + 4, 8), (4, (1 << 32) + 8)):
        with pytest.raises(ValueError, match="2\\^31"):
            HF._adapter_args(make(rows, 1), make(2, 8, 1), make(2, N, 8), scale, index, "add_adapters")
    assert HF._adapter_args(make(8, 1), make(2, 8, 1), make(2, 8, 8), scale, index, "add_adapters").rows == 8
