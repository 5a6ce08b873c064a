"""The wait states between instructions that the hand-written statements of the block-scaled kernels have to keep themselves."""
import os
import re
import subprocess

import pytest

from comfyui_amd import _lib
from tests import test_wait_states as W
from tests.test_gemm4w_registers import OBJDUMP, code_objects


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs llvm-objdump")
def test_block_kernels_keep_the_wait_states(tmp_path, monkeypatch):
    monkeypatch.setattr(W, "KERNELS", re.compile(r"(block_gemm8_kernel|block_gemm_kernel|block_stream_kernel)"))
    seen = set()
    for i, obj in enumerate(code_objects(_lib.LIB_PATH)):
        f = tmp_path / f"{i}.o"
        f.write_bytes(obj)
        text = subprocess.run([OBJDUMP, "-d", str(f)], capture_output=True, text=True, check=True).stdout
        for name, body, at in W.kernels(text):
            seen.add(W.KERNELS.search(name).group(1))
            assert not W.violations(body, at), (name, W.violations(body, at)[:5])
    assert len(seen) == 3
