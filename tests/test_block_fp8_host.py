"""e4m3fn Linears with a scale for each block of 128: what the entry points refuse, without a device."""
import ctypes

import pytest
import torch


def lib():
    from comfyui_amd import _lib
    return _lib


def buffers():
    buf = (ctypes.c_char * 8192)()
    p = ctypes.addressof(buf)
    return buf, (p + 255) // 256 * 256


def test_cast_refusals():
    L = lib()
    keep, p = buffers()
    f = L.lib.hdmoe_quant_block_fp8
    assert f(L.W_E4M3FN, p, 1, 128, p, p, 1, None) == L.E_SHAPE
    assert f(L.W_BF16, p, -1, 128, p, p, 1, None) == L.E_SHAPE
    assert f(L.W_BF16, p, 1, 24, p, p, 1, None) == L.E_SHAPE         # K not a multiple of 16
    assert f(L.W_BF16, p, 1, 0, p, p, 1, None) == L.E_SHAPE
    assert f(L.W_BF16, p, 4, 128, p, p, 3, None) == L.E_SHAPE        # scales of a block would overlap the next one's
    assert f(L.W_BF16, p, 2 ** 31, 128, p, p, 2 ** 31, None) == L.E_SHAPE
    assert f(L.W_BF16, None, 1, 128, p, p, 1, None) == L.E_NULL
    assert f(L.W_BF16, p, 1, 128, None, p, 1, None) == L.E_NULL
    assert f(L.W_BF16, p, 1, 128, p, None, 1, None) == L.E_NULL
    assert f(L.W_BF16, p + 2, 1, 128, p, p, 1, None) == L.E_SHAPE    # not on 16 bytes
    assert f(L.W_BF16, None, 0, 128, None, None, 0, None) == 0


def arguments(p, **changes):
    L = lib()
    a = L.BlockArgs()
    w = (L.BlockWeights * 2)(*(L.BlockWeights(p, p, p, p, None) for _ in range(2)))
    a.a_dtype, a.out_dtype, a.E, a.rows, a.K, a.N = L.W_E4M3FN, L.W_BF16, 2, 4, 128, 128
    a.offsets, a.experts = p, w
    a.routed = L.BlockRows(p, p, 4, p, p, 4)
    for k, v in changes.items():
        setattr(a, k, v)
    a.keep = w
    return a


REFUSED = [dict(out_dtype=1), dict(a_dtype=3), dict(E=33), dict(E=-1), dict(rows=-1), dict(K=0), dict(K=136), dict(N=0), dict(N=24), dict(E=0),
           dict(rows_static=-1), dict(rows_static=3, K_static=128, N_static=100), dict(perm=4096, T=3), dict(K=2 ** 20, N=2 ** 12),
           dict(N=2 ** 30, K=16), dict(N=2 ** 22, K=16), dict(N=16, K=2 ** 23)]


@pytest.mark.parametrize("changes", REFUSED)
@pytest.mark.parametrize("which", ["linear", "swiglu"])
def test_contraction_refuses_sizes(which, changes):
    L = lib()
    keep, p = buffers()
    a = arguments(p, **changes)
    f = L.lib.hdmoe_block_linear if which == "linear" else L.lib.hdmoe_block_swiglu
    assert f(ctypes.byref(a), None) == L.E_SHAPE
    assert which.encode() in L.lib.hdmoe_last_error()


@pytest.mark.parametrize("which", ["linear", "swiglu"])
def test_contraction_refuses_pointers(which):
    L = lib()
    keep, p = buffers()
    f = L.lib.hdmoe_block_linear if which == "linear" else L.lib.hdmoe_block_swiglu
    assert f(None, None) == L.E_NULL
    assert f(ctypes.byref(arguments(p, offsets=None)), None) == L.E_NULL
    assert f(ctypes.byref(arguments(p, experts=None)), None) == L.E_NULL
    rows = lambda *v: dict(routed=L.BlockRows(*v))  # noqa: E731
    assert f(ctypes.byref(arguments(p, **rows(None, p, 4, p, p, 4))), None) == L.E_NULL
    assert f(ctypes.byref(arguments(p, **rows(p, None, 4, p, p, 4))), None) == L.E_NULL
    assert f(ctypes.byref(arguments(p, **rows(p, p, 4, None, p, 4))), None) == L.E_NULL
    assert f(ctypes.byref(arguments(p, **rows(p, p, 3, p, p, 4))), None) == L.E_SHAPE     # scale stride below the rows
    assert f(ctypes.byref(arguments(p, **rows(p + 8, p, 4, p, p, 4))), None) == L.E_SHAPE  # not on 16 bytes
    assert f(ctypes.byref(arguments(p, **rows(p, p, 4, p + 8, p, 4))), None) == L.E_SHAPE
    a = arguments(p)
    a.experts[1].scale = None
    assert f(ctypes.byref(a), None) == L.E_NULL
    a = arguments(p)
    a.experts[1].weight = p + 4
    assert f(ctypes.byref(a), None) == L.E_SHAPE
    a = arguments(p, rows_static=1, K_static=128, N_static=128)
    assert f(ctypes.byref(a), None) == L.E_NULL     # no shared weight
    if which == "swiglu":
        assert f(ctypes.byref(arguments(p, **rows(p, p, 4, p, None, 4))), None) == L.E_NULL
        a = arguments(p)
        a.experts[0].weight3 = None
        assert f(ctypes.byref(a), None) == L.E_NULL
    # 16-bit rows: room for their cast where the contraction does not make it, and the same rows for both groups
    many = dict(a_dtype=L.W_BF16, rows=25600, routed=L.BlockRows(p, None, 0, p, p, 25600))
    assert L.lib.hdmoe_block_workspace_bytes(ctypes.byref(arguments(p, **many)), which == "swiglu") == 25600 * 128 + 25600 * 4
    assert f(ctypes.byref(arguments(p, **many)), None) == L.E_WORKSPACE
    assert f(ctypes.byref(arguments(p, **many, workspace=p + 1, workspace_bytes=1 << 20)), None) == L.E_WORKSPACE
    a = arguments(p, a_dtype=L.W_BF16, rows_static=4, K_static=128, N_static=128, fixed=L.BlockRows(p + 256, None, 0, p, p, 4))
    a.shared = ctypes.pointer(a.keep[0])
    assert f(ctypes.byref(a), None) == L.E_SHAPE
    empty = L.BlockArgs()
    empty.a_dtype = L.W_E4M3FN
    assert f(ctypes.byref(empty), None) == 0        # nothing to do


def test_a_linear_of_16_bit_rows_returns_their_type():
    L = lib()
    keep, p = buffers()
    assert L.lib.hdmoe_block_linear(ctypes.byref(arguments(p, a_dtype=L.W_F16)), None) == L.E_SHAPE


def test_struct_layouts_match_what_a_c_compiler_sees(tmp_path):
    import os
    import subprocess
    L = lib()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"hdmoe_block_weights": L.BlockWeights, "hdmoe_block_rows": L.BlockRows, "hdmoe_block_args": L.BlockArgs}
    lines = []
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "hdmoe.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)])
    got = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"


def test_wrappers_refuse():
    """Types and shapes that the tensor wrappers refuse before they look for a device; a host tensor where one is needed."""
    from comfyui_amd import functional as HF
    F8 = torch.float8_e4m3fn
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    w, sw = torch.zeros((128, 128)).to(F8), torch.ones((1, 1))
    off = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP device"):
        HF.quant_block_fp8(x)
    with pytest.raises(TypeError):
        HF.quant_block_fp8(x.float())
    with pytest.raises(RuntimeError, match="HIP device"):
        HF.linear_block_fp8(x, w, sw)
    with pytest.raises(TypeError, match="out_dtype"):
        HF.linear_block_fp8(x, w, sw, out_dtype=torch.float32)
    with pytest.raises(TypeError, match="scales belong"):
        HF.linear_block_fp8(x, w, sw, scale_x=sw)
    with pytest.raises(ValueError, match="activations"):
        HF.linear_block_fp8(x[None], w, sw)
    with pytest.raises(RuntimeError, match="HIP device"):
        HF.grouped_linear_block_fp8(x, off, [(w, sw, None)])
    with pytest.raises(RuntimeError, match="HIP device"):
        HF.grouped_swiglu_block_fp8(x, off, [(w, sw, w, sw)])
