"""Attention of prompts over 8-bit pages in tiles of 256 (token, head) pairs, against the plain implementation in 64 bits."""
from __future__ import annotations

import pytest
import torch

import plain_few_bits as plain
from test_few_bits_gpu import attention_limit, filled, rand

pytestmark = pytest.mark.gpu


def check(portions, cached, heads, kv, page, span, seed=2, spread=1.0, scale=128 ** -0.5, change=None, pad=8, tokens=None):
    """Portions of prompts behind `cached` keys; a place of the list without a tile; `change` may alter the pages."""
    from inferrs_b200 import kernels as K
    d = 128
    lengths = [c + p for c, p in zip(cached, portions)]
    pages, table = filled(lengths, kv, d, page, seed)
    n = sum(portions)
    q = (spread * rand((n, heads, d), seed + 1)).bfloat16()
    if change is not None:
        change(pages, table, q)
    pos = torch.cat([torch.arange(c, c + p) for c, p in zip(cached, portions)]).int().cuda()
    req = torch.cat([torch.full((p,), i) for i, p in enumerate(portions)]).int().cuda()
    starts = [0]
    for p in portions:
        starts.append(starts[-1] + p)
    tokens = tokens or K.kv8_tile_tokens(heads, kv, d, 1 << 20)
    assert tokens * (heads // kv) > 32
    tile_list = [(i, r) for i in range(len(portions)) for r in range(starts[i], starts[i + 1], tokens)]
    tile_list.insert(1, (-1, 0))
    tile_req, tile_row0 = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in zip(*tile_list))
    q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out = torch.full((n, heads * d + pad), float("nan"), dtype=torch.bfloat16, device="cuda")[:, :heads * d]
    K.paged_attention_kv8(q, pages, table, req, pos, scale, span or None, out, max(lengths), tiles=(tile_req, tile_row0, len(tile_list), q_start, tokens))
    want, weight, size = plain.attention(q, pages.k.double(), pages.v.double(), pages.k_scale.double(), pages.v_scale.double(),
                                         table, req, pos, scale, span)
    limit = attention_limit(want, weight, size, d, max(lengths), torch.bfloat16)
    off = (out.double().view(n, heads, d) - want).abs()
    assert bool((off <= limit).all()), (float((off - limit).max()), int((off > limit).sum()))
    assert K.few_bits_faults() == {}
    return out.view(n, heads, d)


@pytest.mark.parametrize("heads,kv,page", [(8, 2, 16), (32, 8, 16), (4, 4, 48), (20, 4, 64), (32, 2, 128), (6, 2, 16), (40, 1, 32)])
def test_portions_of_every_length(heads, kv, page):
    check((1, 2, 37, 128, 300), (0, 130, 100, 0, 64), heads, kv, page, 0)
    check((257, 64), (1000, 127), heads, kv, page, 0, pad=1)
    check((700,), (0,), heads, kv, page, 0, tokens=max(1, 33 * kv // heads + 1))


@pytest.mark.parametrize("span", [1, 16, 50, 128, 200, 1000, -32, -100, -128])
def test_windows_and_chunks(span):
    check((300, 1, 90), (0, 500, 333), 8, 2, 16, span)
    check((200,), (900,), 32, 4, 32, span, seed=5)


def test_long_contexts():
    check((130, 5), (9000, 4095), 8, 2, 16, 0, seed=3)
    check((2100,), (0,), 4, 1, 16, 0, seed=4)


def test_sharp_and_flat_scores():
    for spread, scale in ((60.0, 128 ** -0.5), (0.0, 128 ** -0.5), (1e-20, 1e18), (1e15, 1e-17), (1.0, -0.2)):
        check((150, 3), (20, 900), 8, 2, 16, 0, seed=7, spread=spread, scale=scale)


@pytest.mark.parametrize("small,great", [(1e-9, 1e9), (1e-24, 1e4), (1e-28, 1e24), (1e-36, 1e36)])
def test_value_scales_far_apart(small, great):
    """Values far smaller than a neighbour's keep their precision where the neighbour is not looked at; the scales of some tiles of
    keys are in the bounds of one exponential a score, of others they are not."""
    def change(pages, table, q):
        at = table[0].long()
        pages.v_scale[at[3], :, 2] *= great
        pages.v_scale[at[5], :, 5] *= small
        pages.v_scale[at[40], :, :] *= small
        loud = pages.k[at[3], 0, 2].float() * pages.k_scale[at[3], 0, 2]
        q[10:, :] = (-8 * loud / loud.norm()).bfloat16()
        q[20:, ::2] = -q[20:, ::2]
    check((250,), (600,), 4, 1, 16, 0, seed=8, scale=3.0, change=change)


def test_vectors_of_zeros_and_pages_that_are_not_there():
    """Zero vectors (scale 0) weigh as any; keys whose page is not in the cache are not seen; a query of zeros takes the mean."""
    from inferrs_b200 import kernels as K

    def change(pages, table, q):
        at = table[0].long()
        for t, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
            t.view(torch.uint8)[at[2]] = 0
            s[at[2]] = 0
        t = pages.v.view(torch.uint8)
        t[at[6], :, 3:9] = 0
        pages.v_scale[at[6], :, 3:9] = 0
        q[5] = 0
    check((140,), (200,), 8, 2, 16, 0, seed=9, change=change)

    # keys of pages that are not there (the plain result from the pages as they were, without those keys)
    pages, table = filled([340], 2, 128, 16, 9)
    q = rand((140, 8, 128), 10).bfloat16()
    pos, req = torch.arange(200, 340, dtype=torch.int32, device="cuda"), torch.zeros(140, dtype=torch.int32, device="cuda")
    lost = table.clone()
    lost[0, 4], lost[0, 9] = -1, pages.k.shape[0]
    row0 = torch.tensor([0, 64, 128], dtype=torch.int32, device="cuda")
    out = torch.empty((140, 1024), dtype=torch.bfloat16, device="cuda")
    K.paged_attention_kv8(q, pages, lost, req, pos, 0.1, None, out, 340,
                          tiles=(torch.zeros_like(row0), row0, 3, torch.tensor([0, 140], dtype=torch.int32, device="cuda"), 64))
    j = torch.arange(340)
    of = table[0].long().cpu()[j // 16]
    k, v = ((t.cpu().double() * s.cpu().double().unsqueeze(-1))[of, :, j % 16].repeat_interleave(4, dim=1)
            for t, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
    seen = (j[None, :] <= pos.cpu()[:, None]) & ~((j // 16 == 4) | (j // 16 == 9))[None, :]
    scores = torch.einsum("rhd,jhd->rhj", q.cpu().double(), k) * 0.1
    weights = torch.softmax(scores.masked_fill(~seen[:, None, :], float("-inf")), dim=-1)
    want, weight = torch.einsum("rhj,jhd->rhd", weights, v), torch.einsum("rhj,jhd->rhd", weights, v.abs())
    size = torch.einsum("rhd,jhd->rhj", q.cpu().double().abs(), k.abs()).amax(dim=-1, keepdim=True) * 0.1
    limit = attention_limit(want, weight, size, 128, 340, torch.bfloat16)
    assert bool(((out.cpu().double().view(140, 8, 128) - want).abs() <= limit).all())
    # rows that see nothing at all
    pages, table = filled([300], 2, 128, 16, 1)
    table.fill_(-1)
    q = rand((70, 8, 128), 4).bfloat16()
    pos, req = torch.arange(230, 300, dtype=torch.int32, device="cuda"), torch.zeros(70, dtype=torch.int32, device="cuda")
    one = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    out = torch.full((70, 1024), float("nan"), dtype=torch.bfloat16, device="cuda")
    K.paged_attention_kv8(q, pages, table, req, pos, 0.1, None, out, 300,
                          tiles=(torch.zeros_like(one), one, 2, torch.tensor([0, 70], dtype=torch.int32, device="cuda"), 64))
    assert bool((out == 0).all())


def test_keys_and_values_that_are_no_numbers():
    """A vector that holds an infinity reads back as none: who sees it gets none, who does not keeps its result."""
    from inferrs_b200 import kernels as K
    pages, table = filled([300], 2, 128, 16, 1)
    at = int(table[0, 12])
    pages.v_scale[at, 0, 8] = float("nan")      # key 200 of the first key/value head
    pages.k_scale[at, 1, 8] = float("nan")
    q = rand((150, 8, 128), 4).bfloat16()
    pos, req = torch.arange(150, 300, dtype=torch.int32, device="cuda"), torch.zeros(150, dtype=torch.int32, device="cuda")
    row0 = torch.tensor([0, 64, 128], dtype=torch.int32, device="cuda")
    out = torch.zeros((150, 1024), dtype=torch.bfloat16, device="cuda")
    K.paged_attention_kv8(q, pages, table, req, pos, 0.1, None, out, 300,
                          tiles=(torch.zeros_like(row0), row0, 3, torch.tensor([0, 150], dtype=torch.int32, device="cuda"), 64))
    assert bool(out[:50].isfinite().all()) and bool(out[50:].isnan().all())


def test_same_bits_again_and_next_to_other_requests():
    a = check((300,), (40,), 8, 2, 16, 0, seed=11)
    b = check((300,), (40,), 8, 2, 16, 0, seed=11)
    assert torch.equal(a, b)


def test_refusals_of_tiles():
    from inferrs_b200 import kernels as K
    pages, table = filled([64], 2, 128, 16, 1)
    q = rand((64, 8, 128), 4).bfloat16()
    pos, req = torch.arange(64, dtype=torch.int32, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda")
    one, start = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    out = torch.empty((64, 1024), dtype=torch.bfloat16, device="cuda")
    for tiles in ((one, one, 1, start, 65), (one, one, 1, start, 0), (one, one, 2, start, 64), (one.long(), one, 1, start, 64),
                  (one, one, 1, start.cpu(), 64)):
        with pytest.raises(K.KernelError):
            K.paged_attention_kv8(q, pages, table, req, pos, 0.1, None, out, 64, tiles=tiles)
    assert K.kv8_tile_tokens(8, 2, 64, 1 << 20) == 8 and K.kv8_tile_tokens(8, 2, 128, 64) == 8 and K.kv8_tile_tokens(8, 2, 128, 1 << 20) == 64


@pytest.mark.parametrize("most", [3, 10, 12, 40])
def test_value_scales_of_every_size(most):
    """Scales spread evenly (in their logarithm) over 2^-most .. 1: around what 32 keys may differ by to share a power of two."""
    def change(pages, table, q):
        pages.v_scale.mul_(torch.exp2(-most * torch.rand(pages.v_scale.shape, generator=torch.Generator(device="cuda").manual_seed(most), device="cuda")))
    check((200,), (300,), 8, 2, 16, 0, seed=12, change=change, scale=0.5)
