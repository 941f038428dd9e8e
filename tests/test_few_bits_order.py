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
