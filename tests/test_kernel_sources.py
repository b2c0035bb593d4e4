"""What the compiler does not look after inside inline assembly, checked in the kernels' sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "origindl_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")))


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_a_write_of_m0_and_a_load_into_lds_are_one_wait_state_apart(path):
    """gfx9 requires one wait state between a scalar write of m0 and an instruction that takes its LDS address from it."""
    text = open(path).read()
    for block in re.findall(r'asm\s*(?:volatile)?\s*\(((?:\s*"(?:[^"\\]|\\.)*")+)', text):
        lines = [l.strip() for l in "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', block)).replace("\\t", "").split("\\n")]
        for i, line in enumerate(lines):
            if re.match(r"s_\w+ m0\b", line):
                assert i + 1 < len(lines) and lines[i + 1].startswith("s_nop"), (os.path.basename(path), line)
