"""Infinities and no numbers in an 8-bit cache: who sees such a vector gets no number, who does not keeps its result."""
from __future__ import annotations

import pytest
import torch

import plain_few_bits as plain
from test_few_bits_gpu import DT, attention_limit, filled, rand, table_for

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


def attend(form, q, pages, table, pos, req, scale, span):
    """Rows one by one, or in tiles of the size that the name says."""
    from inferrs_b200 import kernels as K
    n, heads, d = q.shape
    out, tiles = torch.zeros((n, heads * d), dtype=q.dtype, device="cuda"), None
    if form != "rows":
        tokens = K.kv8_tile_tokens(heads, pages.k.shape[1], d, 1 << 20 if form == "large tiles" else 0)
        row0 = torch.arange(0, n, tokens, dtype=torch.int32, device="cuda")
        tiles = torch.zeros_like(row0), row0, row0.numel(), torch.tensor([0, n], dtype=torch.int32, device="cuda"), tokens
    K.paged_attention_kv8(q, pages, table, req, pos, scale, span or None, out, n, tiles=tiles)
    assert K.few_bits_faults() == {}
    return out.view(n, heads, d)


def seen_by(n, kv, heads, bad, span):
    """[n, heads]: whether a row's head sees one of the vectors (token, key/value head)."""
    sees = torch.zeros((n, heads), dtype=torch.bool, device="cuda")
    for token, head in bad:
        for r in range(token, n):
            if plain.first_visible(r, span) <= token:
                sees[r, head * (heads // kv):(head + 1) * (heads // kv)] = True
    return sees


def check(got, sees, q, pages, table, pos, req, scale, span):
    want, weight, size = plain.attention(q, pages.k.double(), pages.v.double(), pages.k_scale.double(), pages.v_scale.double(), table, req, pos, scale, span)
    near = (got.double() - want).abs() <= attention_limit(want, weight, size, q.shape[2], q.shape[0], q.dtype)
    assert bool(near[~sees].all()) and not bool(near[sees].all(-1).any())


FORMS = [("bf16", 64, "rows"), ("bf16", 64, "tiles"), ("bf16", 128, "rows"), ("bf16", 128, "tiles"), ("bf16", 128, "large tiles"),
         ("bf16", 256, "rows"), ("bf16", 256, "tiles"), ("f32", 128, "rows"), ("bf16", 80, "rows")]


@pytest.mark.parametrize("span", [0, 9, -16])
@pytest.mark.parametrize("dtype,d,form", FORMS)
def test_attention_over_what_was_stored(dtype, d, form, span):
    """Keys and values with infinities of both signs and without numbers; queries of both signs meet each of them."""
    for part in "kv":
        bad = [b for b in BAD if b[0] == part]
        q, pages, table, pos, req = stored(200, 8, 2, d, dtype, 0, False, False, bad)
        q[:, ::2] = -q[:, 1::2]
        got = attend(form, q, pages, table, pos, req, 0.2, span)
        sees = seen_by(200, 2, 8, {(b[1], b[2]) for b in bad}, span)
        assert bool(got[sees].isnan().all())
        check(got, sees, q, pages, table, pos, req, 0.2, span)


@pytest.mark.parametrize("span", [0, 9, -16])
@pytest.mark.parametrize("dtype,d,form", FORMS)
@pytest.mark.parametrize("what", ["key scale", "key code", "value scale", "value code"])
def test_attention_over_pages_that_others_have_filled(what, dtype, d, form, span):
    """Infinite scales, and codes that are no numbers beside a scale that is one."""
    from inferrs_b200 import kernels as K
    pages, table = filled([200], 2, d, 16, 3)
    q = rand((200, 8, d), 4).to(DT[dtype])
    q[:, ::2] = -q[:, 1::2]
    pos, req = torch.arange(200, dtype=torch.int32, device="cuda"), torch.zeros(200, dtype=torch.int32, device="cuda")
    bad = {(3, 0), (40, 1), (41, 0), (130, 0)}
    codes, scales = (pages.k, pages.k_scale) if what.startswith("key") else (pages.v, pages.v_scale)
    for i, (token, head) in enumerate(sorted(bad)):
        at = int(table[0, token // 16]), head, token % 16
        if what.endswith("scale"):
            scales[at] = INF
        else:
            codes.view(torch.uint8)[at][7 * i:7 * i + 2] = torch.tensor([0x7F, 0xFF], dtype=torch.uint8, device="cuda")
    got = attend(form, q, pages, table, pos, req, 0.2, span)
    sees = seen_by(200, 2, 8, bad, span)
    if what.startswith("key"):
        assert bool(got[sees].isnan().all())
    elif what == "value scale":
        assert not bool(got[sees].isfinite().any())
    else:
        assert not bool(got[sees].isfinite().all(-1).any())
    check(got, sees, q, pages, table, pos, req, 0.2, span)
