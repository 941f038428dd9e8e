"""Attention of drafted tokens whose keys are cut into slices (csrc/attention_tree_tcgen05.cu), restated: where a CTA of two sets of rows
puts the sums of its rows, and which CTAs have a slice at all.  No GPU."""
from __future__ import annotations

import os
import random
import re

import pytest

import inferrs_b200

KEYS, ROWS, SLICE, SMEM = 128, 128, 24, 232448
SOURCE = os.path.join(os.path.dirname(inferrs_b200.__file__), "csrc", "attention_tree_tcgen05.cu")


def kernel() -> str:
    with open(SOURCE, encoding="utf-8") as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    return code.split("tree_kernel(const __grid_constant__ CUtensorMap map_k", 1)[1].split("\n}\n", 1)[0]


def leaves_without_a_slice() -> bool:
    """Whether a CTA that no slice is left for returns before it takes tensor memory, by the number of slices behind the first keys."""
    body = kernel()
    found = re.search(r"if \(part >= slices_of\(\(S\.keys \+ KEYS - 1\) / KEYS - t0, slices\)\) return;", body)
    return found is not None and found.start() < body.index("tcgen05.alloc") and "none" not in body


def slices_of(tiles: int, most: int) -> int:
    return max(1, min(most, -(-tiles // SLICE)))


def reach(d: int, rows: int, keys: int, lo_min: int, slices: int, leaves: bool):
    """The end of what the CTAs of these rows write to their shared memory, of those that do."""
    tiles = -(-keys // KEYS) - lo_min // KEYS
    parts = slices_of(tiles, slices)
    top = 0
    for part in range(slices):
        if part >= parts and leaves:
            continue
        if not leaves and part > 0 and part * SLICE * KEYS >= keys:
            continue
        if parts == 1:            # the sums go to the CTA's own shared memory, `most` rows for each of `parts` CTAs
            top = max(top, ((part * rows + rows - 1) * (d + 4) + d) * 4)
    return top


@pytest.mark.parametrize("d", [64, 128])
def test_no_cta_writes_behind_its_shared_memory(d):
    leaves, rng = leaves_without_a_slice(), random.Random(d)
    cases = [(256, 8192 + 64 + more, 8192) for more in (0, 8, 100)]          # chunks of 8,192, contexts shortly behind the second one's start
    for _ in range(2000):
        keys = rng.randrange(1, 200000)
        cases.append((rng.randrange(129, 257), keys, rng.randrange(0, keys + 1)))
    stages = 5 if d == 128 else 8
    tiles = (2 + stages) * d // 64 * ROWS * 128           # the queries and the ring: the sums take their place, barriers stand behind them
    assert tiles + 1024 + 256 <= SMEM
    for rows, keys, lo_min in cases:
        assert reach(d, rows, keys, lo_min, 64, leaves) <= tiles, (rows, keys, lo_min)


def test_a_slice_is_left_for_every_cta_that_stays():
    """The kernel's cut of the tiles: every tile belongs to one CTA, and none of those that stay is without one."""
    rng = random.Random(3)
    for _ in range(2000):
        tiles, slices = rng.randrange(1, 3000), rng.randrange(1, 65)
        parts = slices_of(tiles, slices)
        cuts = [tiles * p // parts for p in range(parts + 1)]
        assert cuts[0] == 0 and cuts[-1] == tiles and all(a < b for a, b in zip(cuts, cuts[1:]))
