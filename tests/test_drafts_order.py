"""Where the kernels for drafted tokens and log probabilities ask that a warp arrives as one, from their sources: the aligned forms want it, and
behind branches and loops that some threads leave early only __syncwarp says so."""
from __future__ import annotations

import os
import re

import inferrs_b200

CSRC = os.path.join(os.path.dirname(inferrs_b200.__file__), "csrc")
FILES = ("attention_tree.cu", "attention_tree_tcgen05.cu", "log_probs.cu", "tree.cuh", "clusters.cuh")


def source(name: str) -> str:
    with open(os.path.join(CSRC, name), encoding="utf-8") as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_barriers_of_a_cluster_meet_whole_warps():
    seen = 0
    for name in FILES:
        lines = [line for line in source(name).split("\n") if line.strip()]
        for i, line in enumerate(lines):
            if "barrier.cluster.arrive" in line:
                assert "__syncwarp();" in lines[i - 1], (name, line)
                seen += 1
    assert seen >= 1


def test_tensor_memory_is_read_by_whole_warps():
    body = source("attention_tree_tcgen05.cu").split("tree_kernel(", 1)[1].split("\n}\n", 1)[0]
    # loops in which some threads skip what comes behind the load
    loops = [loop for loop in re.findall(r"for \([^\n]*\{\n(?:(?!for \()[^\n]*\n){1,3}?[^\n]*tmem_ld32\([^\n]*\n[^\n]*continue;", body)]
    assert len(loops) == 2 and all("__syncwarp();" in loop for loop in loops)
    # one lane tells the products that a half of P is there, and the warp goes on to read the other half
    hand_over = body.split("auto hand_over", 1)[1].split("};", 1)[0].strip().split("\n")
    assert "mbar_arrive" in hand_over[-2] and hand_over[-1].strip() == "__syncwarp();"
