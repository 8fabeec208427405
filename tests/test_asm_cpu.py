"""Inline assembly in csrc/: a block that writes m0, which the compiler uses itself, names it as clobbered."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adafactor-8bit_amd", "csrc")


def test_writes_of_m0_are_named():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        with open(path) as f:
            text = f.read()
        for block in re.findall(r"\basm\b(?:\s+volatile)?\s*\((.*?)\)\s*;", text, re.S):
            if re.search(r"\bs_\w+ m0\b", block):
                seen += 1
                assert '"m0"' in block.split(":")[-1], (os.path.basename(path), block)
    assert seen
