"""A result that lies over the scales or the index of its call, which blocks read after others have written, is refused."""
import ctypes

import pytest

from comfyui_amd import _lib


@pytest.mark.parametrize("name,bytes_", [("scale", 2 * 4), ("index", 64 * 4)])
def test_refused(name, bytes_):
    buf = (ctypes.c_char * (1 << 20))()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    a = _lib.AdapterArgs()
    a.dtype, a.rows, a.requests, a.K, a.N, a.n, a.R = _lib.T_BF16, 64, 64, 256, 256, 2, 16
    for i, n in enumerate(("x", "a", "b", "base", "out", "scale", "index", "workspace")):      # 32 KB each at most, but for the workspace
        setattr(a, n, p + i * (1 << 16))
    a.workspace_bytes = 1 << 17
    result = 64 * 256 * 2
    for at in (a.out, a.out + result - 4, a.out - bytes_ + 4):
        setattr(a, name, at)
        assert _lib.lib.hdmoe_add_adapters(ctypes.byref(a), None) == _lib.E_SHAPE and b"overlaps" in _lib.lib.hdmoe_last_error()
