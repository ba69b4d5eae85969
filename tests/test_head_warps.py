"""Loads of tensor memory and barriers of a cluster take whole warps: the kernel that scores a head's rows
brings its lanes together ahead of each, whatever the code before has left behind."""
import os
import re

from mormot2_ai_b200.csrc import build


def lines_of(name):
    path = os.path.join(os.path.dirname(build.__file__), name)
    with open(path) as f:
        code = [re.sub(r"//.*", "", line).strip() for line in f]
    return [line for line in code if line]


def test_whole_warps():
    code = lines_of("head_scores.cu")
    whole = re.compile(r"TMEM_LD16\(|tmem_ld|cluster_sync_all\(\)")
    found = 0
    for i, line in enumerate(code):
        if not whole.search(line) or whole.search(code[i - 1]):
            continue
        found += 1
        # nothing that a lane may leave alone stands between
        before = [b for b in code[i - 2:i] if b != "tc_fence_before_sync();"]
        assert before[-1] == "__syncwarp();", (i, before, line)
    assert found == 3
