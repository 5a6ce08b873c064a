"""The router's balance loss without a device: the 64-bit formulas against autograd and differences, refusals, the structure."""
import ctypes
import os
import subprocess

import pytest
import torch

from tests import router64

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def loss_of(x, w, idx, alpha, S, mask, dweight):
    """The definition a sequence at a time, and the chosen scores weighted by dweight."""
    L, E, k = x.shape[0] // S, w.shape[0], idx.shape[1]
    p = torch.softmax(x @ w.t(), 1)
    parts = []
    for s in range(S):
        t = s * L + mask[s * L:(s + 1) * L].nonzero()[:, 0]
        if len(t):
            f = torch.stack([(idx[t] == e).sum() for e in range(E)]).double() * E / (k * len(t))
            parts.append((f * p[t].mean(0)).sum())
    chosen = (torch.gather(p, 1, idx.long()) * dweight)[mask].sum()
    return alpha * torch.stack(parts).mean(), chosen


def test_formulas_against_autograd_and_differences():
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn((30, 12), generator=g, dtype=torch.float64), torch.randn((5, 12), generator=g, dtype=torch.float64)
    idx = torch.randint(0, 5, (30, 2), generator=g)
    mask = torch.rand(30, generator=g) < 0.7
    mask[10:20] = False                       # the second of three sequences holds nothing
    dweight = torch.randn((30, 2), generator=g, dtype=torch.float64)
    dloss = torch.tensor(3.0, dtype=torch.float64)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    loss, chosen = loss_of(*leaves, idx, 0.3, 3, mask, dweight)
    want = torch.autograd.grad(loss * dloss + chosen, leaves)
    (l, _), counts, _, (dx, _), (dw, _) = router64.balance(x, w, idx, 0.3, 3, mask, dloss, dweight)
    assert torch.allclose(l, loss.detach()) and int(counts.sum()) == 2 * int(mask.sum()) and not counts[1].any()
    assert torch.allclose(dx, want[0], rtol=1e-11, atol=1e-12) and torch.allclose(dw, want[1], rtol=1e-11, atol=1e-12)
    h, mx, mw = 1e-6, torch.randn(x.shape, generator=g, dtype=torch.float64), torch.randn(w.shape, generator=g, dtype=torch.float64)

    def along(s):
        a, b = loss_of(x + s * h * mx, w + s * h * mw, idx, 0.3, 3, mask, dweight)
        return a * dloss + b
    told = (dx * mx).sum() + (dw * mw).sum()
    assert abs((along(1) - along(-1)) / (2 * h) - told) < 1e-6 * (1 + abs(told))


def test_refusals():
    from comfyui_amd import functional as HF
    x, w, idx = torch.zeros((4, 16), dtype=torch.bfloat16), torch.zeros((3, 16), dtype=torch.bfloat16), torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        HF.gate_balance(x, w, idx)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        HF.gate_balance(x.float(), w, idx)
    with pytest.raises(RuntimeError, match="no CPU path"):
        HF.gate_balance_backward(torch.ones(()), x, w, idx, torch.zeros((1, 3), dtype=torch.int32), torch.zeros((4, 3)))


def test_library_refusals_without_a_device():
    from comfyui_amd import _lib
    L = _lib.lib
    buf = (ctypes.c_char * 64)()
    ptr = (ctypes.addressof(buf) + 15) // 16 * 16

    def args(**kwargs):
        a = _lib.BalanceArgs()
        a.dtype, a.T, a.sequences, a.D, a.E, a.k, a.alpha = _lib.T_BF16, 4096, 4, 256, 4, 2, 0.01
        for name in ("x", "gate_w", "topk_idx", "scores", "counts", "loss", "dloss", "dweight", "dx", "dgate_w"):
            setattr(a, name, ptr)
        for k, v in kwargs.items():
            setattr(a, k, v)
        return a

    for fn, own in ((L.hdmoe_gate_balance, ("loss",)), (L.hdmoe_gate_balance_backward, ("dloss", "dx", "dgate_w"))):
        assert fn(None, None) == _lib.E_NULL
        for bad in (dict(dtype=_lib.T_F32), dict(T=-1), dict(T=4097), dict(sequences=0), dict(D=0), dict(D=12), dict(E=0), dict(E=17), dict(k=0), dict(k=17)):
            assert fn(ctypes.byref(args(**bad)), None) == _lib.E_SHAPE, bad
        for missing in ("x", "gate_w", "topk_idx", "scores", "counts", *own):
            assert fn(ctypes.byref(args(**{missing: None})), None) == _lib.E_NULL, missing
        backward = fn is L.hdmoe_gate_balance_backward
        need = L.hdmoe_gate_balance_workspace_bytes(ctypes.byref(args()), int(backward))
        assert need > 0
        for ws, size in ((None, 0), (ptr, need - 1), (ptr + 4, need)):
            assert fn(ctypes.byref(args(workspace=ws, workspace_bytes=size)), None) == _lib.E_WORKSPACE
        for bad in (dict(T=1 << 23, sequences=1 << 23), dict(T=1 << 30, sequences=1 << 22)):      # more threads than a launch has
            assert fn(ctypes.byref(args(**bad)), None) == _lib.E_SHAPE, bad
        assert fn(ctypes.byref(args(T=1 << 20, sequences=1 << 20)), None) == _lib.E_WORKSPACE
    masked = L.hdmoe_gate_balance_workspace_bytes(ctypes.byref(args(mask=ptr)), 1)
    assert masked > L.hdmoe_gate_balance_workspace_bytes(ctypes.byref(args()), 1)


def test_struct_layout_matches_what_a_c_compiler_sees(tmp_path):
    from comfyui_amd import _lib
    cname, cls = "hdmoe_balance_args", _lib.BalanceArgs
    lines = [f'printf("{cname} %zu\\n", sizeof({cname}));'] + [f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hdmoe.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = dict(l.split() for l in subprocess.check_output([str(exe)], text=True).splitlines())
    assert int(got[cname]) == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert int(got[f]) == getattr(cls, f).offset, f


def test_sizes_that_a_c_int_does_not_hold(monkeypatch):
    from comfyui_amd import functional as HF
    monkeypatch.setattr(HF, "_need_hip", lambda *a: None)
    make = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    for T, sequences in (((1 << 32) + 4, 1), ((1 << 32) + 4, (1 << 32) + 4)):
        with pytest.raises(ValueError, match="2\\^31"):
            HF._balance_args(make(T, 8), make(4, 8), make(T, 2, dtype=torch.int32), sequences, None, 0.01, "gate_balance")
    assert HF._balance_args(make(64, 8), make(4, 8), make(64, 2, dtype=torch.int32), 2, None, 0.01, "gate_balance").T == 64
