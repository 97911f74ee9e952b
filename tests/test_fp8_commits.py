"""CPU: the source rule of the 8-bit kernels' commits has something to look at.  (tcgen05.commit covers the UMMAs of the thread that
executes it; the rule itself stands in test_fp8_window_arguments.py.)"""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tnn_b200", "csrc")


def _text(path):
    with open(path) as f:
        return re.sub(r"//[^\n]*", "", f.read())


SOURCES = {os.path.basename(f): _text(f) for f in glob.glob(os.path.join(CSRC, "*.cu"))}
EIGHT_BIT = sorted(n for n, t in SOURCES.items() if "umma_f8_ss(" in t)


def _enclosing(text, at):
    depth, i = 0, at
    while depth >= 0:
        i -= 1
        depth += {"}": 1, "{": -1}.get(text[i], 0)
    return text[i:at]


def test_there_are_8_bit_kernels_on_the_tensor_core():
    assert EIGHT_BIT == ["linear_fp8.cu"]


@pytest.mark.parametrize("name", EIGHT_BIT)
def test_their_commits_are_named_and_stand_with_their_ummas(name):
    text = SOURCES[name]
    found = [m.start() for m in re.finditer(r"\bumma_f8_commit\(", text)]
    assert found and not re.search(r"\bumma_commit(_pair)?\(|tcgen05\.commit", text)     # no commit that the rule does not see
    assert all(re.search(r"\bumma_f8_ss\(", _enclosing(text, at)) for at in found)


def test_the_name_is_the_commit_itself():
    text = _text(os.path.join(CSRC, "ptx.cuh"))
    assert re.search(r"void umma_f8_commit\(uint64_t\* bar\) \{ umma_commit\(bar\); \}", text)
    assert len(re.findall(r"\bumma_f8_ss\w*\(", text)) == 1
