"""The package where _block_calls.so is missing or was built for another torch or another library: it imports, with a warning, and makes the calls itself."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import sys, types
{block}
import torch
from comfyui_amd import functional as HF
from comfyui_amd import hidream, hunyuan3d, ops
assert HF._block_calls is None and HF._stream_here(torch.zeros(1)) is None
try:
    HF.quant_block_fp8(torch.zeros((4, 128), dtype=torch.bfloat16))
except RuntimeError as e:
    assert "HIP device" in str(e)
else:
    raise AssertionError
"""
MISSING = "sys.modules['comfyui_amd._block_calls'] = None"
OTHER = "m = types.ModuleType('m'); m.torch_version = '1.0'; sys.modules['comfyui_amd._block_calls'] = m"


OLDER = "import torch; m = types.ModuleType('m'); m.torch_version, m.hdmoe_version = torch.__version__, 117; sys.modules['comfyui_amd._block_calls'] = m"


@pytest.mark.parametrize("block", [MISSING, OTHER, OLDER], ids=["missing", "other torch", "older library"])
def test_import(block):
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(block=block)], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "no compiled calls" in r.stderr


def test_the_built_one_is_taken():
    import torch
    from comfyui_amd import functional as HF
    assert HF._block_calls is not None and HF._block_calls.torch_version == torch.__version__ and HF._block_calls.hdmoe_version == HF.lib.hdmoe_version()
