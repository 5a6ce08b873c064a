"""The package where _row_calls.so is missing or was built for another torch or another library: it imports, with a warning, and makes the calls itself."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import sys, types
import torch
{block}
from comfyui_amd import autograd, functional as HF
assert HF._row_calls is None
x = torch.zeros((4, 128), dtype=torch.bfloat16)
for call in (lambda: HF.layer_norm(x), lambda: autograd.layer_norm(x)):
    try:
        call()
    except RuntimeError as e:
        assert "HIP device" in str(e)
    else:
        raise AssertionError
"""
BLOCKS = {"missing": "sys.modules['comfyui_amd._row_calls'] = None",
          "other torch": "m = types.ModuleType('m'); m.torch_version = '1.0'; sys.modules['comfyui_amd._row_calls'] = m",
          "older library": "m = types.ModuleType('m'); m.torch_version, m.hdmoe_version = torch.__version__, 118; sys.modules['comfyui_amd._row_calls'] = m"}


@pytest.mark.parametrize("block", list(BLOCKS))
def test_import(block):
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(block=BLOCKS[block])], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "no compiled calls of the layer norm" in r.stderr


def test_the_built_one_is_taken():
    import torch
    from comfyui_amd import functional as HF
    assert HF._row_calls is not None and HF._row_calls.torch_version == torch.__version__ and HF._row_calls.hdmoe_version == HF.lib.hdmoe_version()
