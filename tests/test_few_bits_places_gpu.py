"""Tensors of the operators in few bits that start anywhere in memory, lists that say less than they should, rows of nobody."""
from __future__ import annotations

import pytest
import torch

from test_few_bits_gpu import rand, table_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4, 6])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_queries_go_anywhere(d, offset):
    """Queries (and the projection's rows) on 2, 4 and 8 bytes, as parts of a larger piece of memory.  The kernels for whole heads and for any
    tensors round a query once, from sums of their own order: a place of bfloat16 apart at most."""
    from inferrs_b200 import kernels as K
    n, heads, kv = 70, 4, 2
    table, n_pages = table_for([n], 16, 1)
    qkv = rand((n, (heads + 2 * kv) * d), 2).bfloat16()
    weight = (1 + 0.1 * rand((d,), 3)).bfloat16()
    angle = 3 * rand((n, d // 2), 4)
    pos, req = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")

    def store(rows, q):
        pages = K.Kv8Pages.zeros(n_pages, kv, 16, d, "cuda")
        K.qk_norm_rope_store_kv8(rows, heads, kv, d, weight, weight, 1e-6, angle.cos(), angle.sin(), d, pos, req, table, pages, q)
        return pages

    want = torch.empty((n, heads, d), dtype=torch.bfloat16, device="cuda")
    same = store(qkv, want)
    room = torch.full((n * heads * d + 8,), 7.0, dtype=torch.bfloat16, device="cuda")
    got = room[offset:offset + n * heads * d].view(n, heads, d)
    pages = store(qkv, got)
    assert bool(((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -20).all())
    assert bool((room[:offset] == 7).all()) and bool((room[offset + n * heads * d:] == 7).all())
    assert torch.equal(pages.v.view(torch.uint8), same.v.view(torch.uint8)) and torch.equal(pages.v_scale, same.v_scale)
    shifted = torch.empty((qkv.numel() + 8,), dtype=torch.bfloat16, device="cuda")
    rows = shifted[offset:offset + qkv.numel()].view_as(qkv)
    rows.copy_(qkv)
    again = torch.empty_like(want)
    store(rows, again)
    assert bool(((again.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -20).all())
