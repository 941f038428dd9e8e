"""Tensors of the operators in few bits that start anywhere in memory, lists that say less than they should, rows of nobody."""
from __future__ import annotations

import pytest
import torch

import plain_few_bits as plain
from test_few_bits_gpu import DT, attention_limit, filled, rand, table_for

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


@pytest.mark.parametrize("tokens", [8, 64])
def test_tiles_of_requests_that_are_not_there(tokens):
    """A list of starts that is too short, or a number of tiles that is none, is refused; a tile of a request beyond the table's is no tile."""
    from inferrs_b200 import kernels as K
    pages, table = filled([64, 64], 2, 128, 16, 1)
    q, out = rand((128, 8, 128), 4).bfloat16(), torch.full((128, 1024), 7.0, dtype=torch.bfloat16, device="cuda")
    numbers = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    pos, req = torch.arange(64, dtype=torch.int32, device="cuda").repeat(2), torch.arange(2, dtype=torch.int32, device="cuda").repeat_interleave(64)
    tile_req, tile_row0, starts = numbers(0, 2, 5, -1, 1), numbers(0, 64, 64, 64, 64), numbers(0, 64, 128)

    def call(n_tiles=5, starts=starts):
        K.paged_attention_kv8(q, pages, table, req, pos, 0.1, None, out, 64, tiles=(tile_req, tile_row0, n_tiles, starts, tokens))

    for bad in (dict(starts=starts[:2]), dict(starts=starts[:0]), dict(n_tiles=6), dict(n_tiles=-1)):
        with pytest.raises(K.KernelError):
            call(**bad)
    codes, scales = [t.double() for t in (pages.k, pages.v)], [t.double() for t in (pages.k_scale, pages.v_scale)]
    want, weight, size = plain.attention(q, *codes, *scales, table, req, pos, 0.1, 0)
    limit = attention_limit(want, weight, size, 128, 64, torch.bfloat16)

    def right():                               # of every row
        return ((out.double().view(128, 8, 128) - want).abs() <= limit).all(-1).all(-1)

    call(4)                                    # the first request's first tile alone
    assert bool(right()[:tokens].all()) and bool((out[tokens:] == 7).all())
    call()
    assert bool(right()[64:64 + tokens].all())
    assert K.few_bits_faults() == {}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_no_request_get_zeros(dtype):
    """Rows whose request is -1, or beyond the table's, beside rows of requests."""
    from inferrs_b200 import kernels as K
    pages, table = filled([300, 64, 5], 2, 128, 16, 1)
    q = rand((5, 8, 128), 4).to(DT[dtype])
    pos = torch.tensor([299, 40, 63, 17, 4], dtype=torch.int32, device="cuda")
    req = torch.tensor([0, -1, 1, 3, 2], dtype=torch.int32, device="cuda")
    out, real = (torch.full((5, 1024), 7.0, dtype=DT[dtype], device="cuda") for _ in range(2))
    K.paged_attention_kv8(q, pages, table, req, pos, 0.1, None, out, 300)
    K.paged_attention_kv8(q, pages, table, req.clamp(0, 2), pos, 0.1, None, real, 300)
    assert bool((out[[1, 3]] == 0).all())
    assert torch.equal(out[[0, 2, 4]], real[[0, 2, 4]])


def test_matrices_and_rows_on_different_devices_are_refused():
    """Said by the matrix's device alone (nothing is launched)."""
    from inferrs_b200 import kernels as K
    x, out = rand((4, 64), 1), torch.empty((4, 4), device="cuda")
    here, there = K.quantize_mx4(x), K.quantize_mx4(x)
    there.device = torch.device("cuda", 1)
    for call in (lambda: K.quantize_mx4(x, there), lambda: K.dequantize_mx4(there, torch.empty_like(x)), lambda: K.linear_mx4(x, there, out),
                 lambda: K.linear_mx4(there, here, out)):
        with pytest.raises(K.KernelError):
            call()
    K.linear_mx4(x, here, out)
    K.linear_mx4(here, here, out)
    K.dequantize_mx4(here, torch.empty_like(x))
    assert K.quantize_mx4(x, here) is here


@pytest.mark.parametrize("n_pages,kv,page,d", [(1, 1, 1, 4), (3, 1, 1, 12), (5, 3, 1, 20), (7, 1, 3, 4)])
def test_pages_of_any_size_and_number(n_pages, kv, page, d):
    """Keys and values start on 16 bytes whatever the pages before them take; a token in the last place is found again."""
    from inferrs_b200 import kernels as K
    pages = K.Kv8Pages.zeros(n_pages, kv, page, d, "cuda")
    table = torch.arange(n_pages, dtype=torch.int32, device="cuda").view(1, -1)
    qkv, q = rand((1, 3 * kv * d), 1), torch.empty((1, kv, d), device="cuda")
    pos, req = torch.tensor([n_pages * page - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    K.qk_norm_rope_store_kv8(qkv, kv, kv, d, None, None, 0.0, None, None, 0, pos, req, table, pages, q)
    out = torch.empty((1, kv * d), device="cuda")
    K.paged_attention_kv8(q, pages, table, req, pos, 1.0, 1, out, n_pages * page)      # a window of one key: its value
    value = qkv.view(3, kv, d)[2]
    assert bool(((out.view(kv, d) - value).abs() <= value.abs() * 2.0 ** -4 + value.abs().amax(-1, keepdim=True) * 2.0 ** -17).all())
