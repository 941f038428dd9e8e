"""The barriers of the product of few rows with 4-bit weights (csrc/gemm_mx4.cu), restated: one thread brings weights, helper warps
bring scales and pieces to every helpers-th stage, one thread multiplies; a wait knows a barrier's phase by its parity alone."""
from __future__ import annotations

import random

import pytest


def run(stages: int, blocks: int, helpers: int, seed: int) -> str:
    rng = random.Random(seed)
    arrivals, full, empty = [2] * stages, [0] * stages, [0] * stages      # arrivals still missing, completed phases
    filled = [[False, False] for _ in range(blocks)]
    brought = multiplied = 0
    at = list(range(helpers))

    def free(i):          # the wait for the place of block i, as the kernel asks for it
        return i < stages or (empty[i % stages] & 1) != ((i // stages - 1) & 1)

    for _ in range(100 * blocks * (helpers + 2)):
        if multiplied == blocks:
            return "done"
        who = rng.randrange(2 + helpers)
        if who == 0 and brought < blocks and free(brought):
            i, part = brought, 0
            brought += 1
        elif who >= 2 and at[who - 2] < blocks and free(at[who - 2]):
            i, part = at[who - 2], 1
            at[who - 2] += helpers
        else:
            if who == 1 and (full[multiplied % stages] & 1) != ((multiplied // stages) & 1):
                if filled[multiplied] != [True, True]:
                    return "multiplied before it was there"
                empty[multiplied % stages] += 1
                multiplied += 1
            continue
        s = i % stages
        if full[s] != i // stages or filled[i][part]:
            return "filled before the place was free"
        filled[i][part] = True
        arrivals[s] -= 1
        if arrivals[s] == 0:
            arrivals[s], full[s] = 2, full[s] + 1
    return "stuck"


@pytest.mark.parametrize("stages", range(1, 10))
def test_no_wait_passes_before_its_time(stages):
    helpers = min(4, stages)
    assert {run(stages, blocks, helpers, seed) for blocks in (1, 2, 3, 5, 8, 13, 40) for seed in range(40)} == {"done"}


def test_more_helpers_than_stages_would_mistake_one_phase_for_another():
    assert "filled before the place was free" in {run(3, 32, 4, seed) for seed in range(40)}
