"""Rules of PTX that no compiler and no run tells: checked in the kernels' sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blog_b200", "csrc")
SOURCES = sorted(p for p in glob.glob(os.path.join(CSRC, "*.cu")) if "reg_dec<" in open(p).read())


def _conditions(text, at):
    """The conditions on `warp` that the statement at `at` stands under, those of the branches before its own among them."""
    blocks, start, closed = [], 0, ""  # open blocks: what stood before each of their braces and of the chain's earlier ones
    for i in range(at):
        c = text[i]
        if c == "{":
            head = text[start:i]
            blocks.append((closed if re.match(r"\s*else\b", head) else "") + head)
            start = i + 1
        elif c == "}":
            closed, start = blocks.pop(), i + 1
        elif c == ";":
            start = i + 1
    return re.findall(r"\bwarp\s*(==|!=|<=|>=|<|>|%|&)\s*(\w+)", " ".join(blocks) + text[start:at])


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_warps_of_a_group_change_their_registers_together(path):
    """setmaxnreg is for all four warps of a warpgroup: no condition on the way to one tells them apart."""
    text = re.sub(r"//[^\n]*|\"[^\"\n]*\"", "", open(path).read())
    value = {k: int(v) for k, v in re.findall(r"\b(k\w+) = (\d+)[,;]", text)}
    calls = list(re.finditer(r"\breg_(?:inc|dec)<\w+>\(\)", text))
    assert len(calls) >= 3
    for call in calls:
        for op, n in _conditions(text, call.start()):
            n = int(n) if n.isdigit() else value[n]
            assert op in ("<", ">=") and n % 4 == 0, (text.count("\n", 0, call.start()) + 1, op, n)
