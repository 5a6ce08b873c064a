"""What the hand-written statements of the block-scaled kernels change is named to the compiler, which sets m0 for LDS loads of its own."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def statements():
    """asm statements of blockscale.hip, from their opening bracket to the closing one."""
    text = open(os.path.join(ROOT, "comfyui_amd", "csrc", "blockscale.hip")).read()
    for at in re.finditer(r"asm volatile\(", text):
        depth, i, quoted = 1, at.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[at.end():i - 1]


def test_m0_is_named_where_it_is_written():
    writers = [s for s in statements() if re.search(r"s_\w+ m0\b", s) or s.lstrip().startswith("TEXT")]
    assert len(writers) >= 5      # the loads to LDS, and the K loop, whose text is generated
    assert [s for s in writers if '"m0"' not in s.rsplit(":", 1)[1]] == []


def test_the_generated_loop_writes_only_what_the_statement_names():
    """Scalar registers of the K loop: operands by name, and the ones among the clobbers."""
    from comfyui_amd.csrc import gen_block_fp8 as G
    (loop,) = [s for s in statements() if s.lstrip().startswith("TEXT")]
    named = set(re.findall(r'"(\w+)"', loop.rsplit(":", 1)[1]))
    for gate_up in (False, True):
        for line in G.tile(gate_up):
            m = re.match(r"s_(?:add|sub|mov|cselect|lshl|or|and)\w* ([^,]+),", line)
            if m and not m.group(1).startswith("%["):
                assert m.group(1) in named, line
            if line.startswith("s_cmp"):
                assert "scc" in named
