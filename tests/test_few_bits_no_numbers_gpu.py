"""Infinities and no numbers in an 8-bit cache: who sees such a vector gets no number, who does not keeps its result."""
from __future__ import annotations

import pytest
import torch

from test_few_bits_gpu import DT, rand, table_for

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def stored(n, heads, kv, d, dtype, rot, interleaved, norm, bad, seed=1):
    """One request's n tokens in a cache: (queries, pages, table, positions, requests); bad: (part, token, head, place, number)."""
    from inferrs_b200 import kernels as K
    table, n_pages = table_for([n], 16, seed)
    qkv = rand((n, heads + 2 * kv, d), seed + 1).to(DT[dtype])
    for part, token, head, place, number in bad:
        qkv[token, heads + (kv if part == "v" else 0) + head, place] = number
    weight = (1 + 0.1 * rand((d,), seed + 2)).to(DT[dtype]) if norm else None
    angle = 3 * rand((n, max(rot // 2, 1)), seed + 3)
    cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
    pos, req = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    q, pages = torch.empty((n, heads, d), dtype=DT[dtype], device="cuda"), K.Kv8Pages.zeros(n_pages, kv, 16, d, "cuda")
    K.qk_norm_rope_store_kv8(qkv.view(n, -1), heads, kv, d, weight, weight, 1e-6, cos, sin, rot, pos, req, table, pages, q,
                             interleaved=interleaved)
    return q, pages, table, pos, req


BAD = [("k", 3, 0, 5, INF), ("k", 40, 1, 0, -INF), ("k", 41, 0, 7, NAN), ("v", 50, 1, 3, INF), ("v", 52, 0, 11, NAN), ("v", 52, 0, 8, -INF)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,rot,interleaved,norm", [(128, 128, False, False), (64, 64, False, True), (256, 256, False, False),
                                                    (128, 64, False, False), (64, 64, True, True), (80, 0, False, False), (12, 12, False, False)])
def test_such_a_vector_is_stored_as_zeros_without_a_scale(d, rot, interleaved, norm, dtype):
    """Its scale is no number, its codes are numbers (a product with them would reach keys and rows that are none of its); the others are as without it."""
    _, pages, table, pos, _ = stored(60, 4, 2, d, dtype, rot, interleaved, norm, BAD)
    _, clean, _, _, _ = stored(60, 4, 2, d, dtype, rot, interleaved, norm, [])
    at = table[0].long()[(pos // 16).long()], (pos % 16).long()
    for part, codes, scales, same_codes, same_scales in (("k", pages.k, pages.k_scale, clean.k, clean.k_scale),
                                                         ("v", pages.v, pages.v_scale, clean.v, clean.v_scale)):
        codes, scales, same_codes, same_scales = (t[at[0], :, at[1]] for t in (codes.view(torch.uint8), scales, same_codes.view(torch.uint8), same_scales))
        none = torch.zeros((60, 2), dtype=torch.bool, device="cuda")
        for p, token, head, _, _ in BAD:
            if p == part:
                none[token, head] = True
        assert torch.equal(scales.isnan(), none) and bool((codes[none] == 0).all())
        assert torch.equal(codes[~none], same_codes[~none]) and torch.equal(scales[~none], same_scales[~none])
