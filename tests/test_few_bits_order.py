"""What the kernels in few bits read before the kernels ahead have ended, from their sources: nothing that one of them may write."""
from __future__ import annotations

import os
import re

import inferrs_b200

CSRC = os.path.join(os.path.dirname(inferrs_b200.__file__), "csrc")


def source(name: str) -> str:
    with open(os.path.join(CSRC, name), encoding="utf-8") as f:
        return f.read()


def test_products_wait_for_whoever_may_write_their_weights():
    """A kernel that lets the next one start before it has waited hands the next one's early reads on to what is ahead of it: quantize_mx4,
    the rows' way to pieces and the product start one in the other.  Outside captured steps a product therefore waits before it reads."""
    rules = re.findall(r"\bp\.wait_first = ([^;]+);", source("gemm_mx4.cu"))
    assert len(rules) == 2
    for rule in rules:
        names = set(re.findall(r"[A-Za-z_]\w*", rule))
        for other in (False, True):          # whatever else the rule asks
            said = eval(rule.replace("!", " not ").replace("&&", " and ").replace("||", " or "), {n: n != "ib_pdl_enabled" and other for n in names})
            assert said, rule


def test_no_kernel_reads_ahead_of_its_wait_through_a_restricted_pointer():
    """Loads through a `const __restrict__` parameter may be moved ahead of the wait for the kernels ahead (common.cuh): every kernel of this
    library, all of which start early, takes such a parameter through ib_after_wait, behind a wait, before it uses it."""
    seen = 0
    for name in ("few_bits.cu", "gemm_mx4.cu", "kv8.cu", "attention_kv8.cu", "attention_kv8_prompt.cu"):
        for kernel in source(name).split("__global__ ")[1:]:
            head, body = kernel.split(") {\n", 1)
            body = body.split("\n}\n", 1)[0]
            code = re.sub(r"//[^\n]*", "", body)
            waits = [m.start() for m in re.finditer(r"ib_grid_dependency_(sync|wait)\(\)", code)]
            for pointer in re.findall(r"const \w+\* __restrict__ (\w+)", head):
                taken = code.find(f"{pointer} = ib_after_wait({pointer});")
                used = re.search(rf"\b{pointer}\b", code)
                assert taken >= 0 and used.start() == taken and any(w < taken for w in waits), (name, pointer)
                seen += 1
    assert seen >= 20


def test_barriers_of_a_cluster_meet_whole_warps():
    """The aligned forms ask that a warp's threads arrive as one; behind loops that some of them leave early only __syncwarp says so."""
    seen = 0
    for name in ("gemm_mx4.cu", "attention_kv8.cu"):
        lines = [line for line in source(name).split("\n") if line.strip() and not line.strip().startswith("//")]
        for i, line in enumerate(lines):
            if "barrier.cluster.arrive.release.aligned" in line:
                assert "__syncwarp();" in lines[i - 1] or "__syncwarp();" in line, (name, line)
                seen += 1
    assert seen >= 2
