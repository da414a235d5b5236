"""Rules that the kernels' sources keep because no run can be relied on to show that they were broken."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpt-neox_amd", "csrc")
SOURCES = sorted(p for kind in ("*.hip", "*.hpp", "*.inl") for p in glob.glob(os.path.join(CSRC, kind)))
ASM = re.compile(r'\basm\b(?:\s+volatile)?\s*\(\s*"([^"]*)"')


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_inline_assembly_holds_no_instruction_that_reads_registers(path):
    # A vector instruction that reads the result of a matrix instruction needs wait states in between.  The compiler puts
    # them before instructions that it knows; what stands in inline assembly would read an unfinished sum.
    with open(path) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    found = ASM.findall(text)
    assert len(found) == len(re.findall(r"\basm\b", text)), "an asm statement that this test cannot read"
    for template in found:
        assert template == "" or re.fullmatch(r"s_waitcnt [a-z]+cnt\(\d+\)", template), template
