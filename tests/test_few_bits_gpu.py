"""4-bit matrices, their products, 8-bit keys and values and attention over them, each against 64 bits."""
from __future__ import annotations

import pytest
import torch

import plain_few_bits as plain

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(shape, seed):
    return torch.randn(shape, generator=gen(seed), device="cuda")


def half_ulp(y, dtype):
    """What rounding to ``dtype`` (8 or 24 significant bits) may move a number by."""
    return y.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) + 1e-38


def apart(x, pad):
    """The same rows, ``pad`` numbers apart."""
    wide = torch.full((x.shape[0], x.shape[1] + pad), float("nan"), dtype=x.dtype, device=x.device)
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


# ---- rows in 4 bits -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,pad", [(1, 1, 0), (1, 32, 0), (3, 33, 0), (129, 127, 1), (5, 128, 8), (130, 129, 0), (31, 257, 0),
                                            (2, 5000, 3), (300, 512, 0), (1000, 96, 0)])
def test_rows_in_four_bits(rows, width, pad, dtype):
    from inferrs_b200 import kernels as K
    x = rand((rows, width), rows + width) * torch.exp(3 * rand((rows, width), 5))
    x = apart(x.to(DT[dtype]), pad) if pad else x.to(DT[dtype])
    want, byte = plain.values4(x)
    w = K.quantize_mx4(x)
    got = plain.scale_bytes(w.scales, rows, width)
    blocks = byte.shape[1]
    assert torch.equal(got[:, :blocks], byte.int())
    assert bool((got[:, blocks:] != 255).all())
    values = plain.code_values(w.codes)
    assert bool((values[:, width:] == 0).all())
    assert torch.equal(values[:, :width] * torch.exp2(byte.double() - 127).repeat_interleave(32, dim=1)[:, :width], want)
    for out_type in DT.values():
        out = apart(torch.zeros((rows, width), device="cuda").to(out_type), pad)
        K.dequantize_mx4(w, out)
        assert torch.equal(out.double(), want.to(out_type).double())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_four_bits_at_ties_ends_of_the_range_and_no_numbers(dtype):
    from inferrs_b200 import kernels as K
    x = torch.zeros((12, 64), device="cuda")
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device="cuda")
    x[0, :8], x[0, 8:16] = ties, -ties                       # every tie, both signs; unit 1
    x[1, 0], x[2, 0], x[3, 0] = 7.0, 7.0625, 7.96875         # up to 7 the unit is 1, beyond it 2
    x[4, :32] = 2.0 ** -126 * 1.5                            # exponents that the scale cannot follow
    x[5, :32] = 2.0 ** -130
    x[6, :4] = 2.0 ** 127 * torch.tensor([1.0, -1.875, 0.5, 0.25], device="cuda")
    x[7, 3], x[8, 3], x[9, 40] = float("inf"), float("nan"), -float("inf")
    x[7:10, 5], x[7:10, 50] = 1.0, 3.0                       # the other block of such a row keeps its numbers
    x[10, 0], x[10, 1] = 1.0, -1e-30
    x = x.to(DT[dtype])
    want, byte = plain.values4(x)
    w = K.quantize_mx4(x)
    assert torch.equal(plain.scale_bytes(w.scales, 12, 64)[:, :2], byte.int())
    out = torch.empty((12, 64), device="cuda")
    K.dequantize_mx4(w, out)
    assert torch.equal(out.double().nan_to_num(12345.0), want.float().double().nan_to_num(12345.0))
    assert bool(out[7, :32].isnan().all()) and float(out[7, 50]) == 3.0 and float(out[9, 5]) == 1.0


def test_quantize_writes_into_a_given_matrix():
    from inferrs_b200 import kernels as K
    x, y = rand((140, 200), 1), rand((140, 200), 2)
    w = K.quantize_mx4(x)
    assert K.quantize_mx4(y, w) is w
    fresh = K.quantize_mx4(y)
    assert torch.equal(w.codes, fresh.codes)
    K.quantize_mx4(torch.empty((0, 64), device="cuda"))
    assert w.bytes() == w.codes.numel() + w.scales.numel() and w.shape == (140, 200)


# ---- products ---------------------------------------------------------------------------------------------------------------
def product_limit(x, w, dtype_in, dtype_out, want):
    """Sums of k numbers in float32, in any order and where an addition may cut instead of round (2^-23 of what has been
    added up, at most k additions a result); bfloat16 rows as pieces: 2^-22 of the largest of a number's block of 32; the
    result's rounding."""
    k = x.shape[1]
    limit = (k + 8) * 2.0 ** -23 * (x.abs() @ w.abs().t())
    if dtype_in == "bf16":
        blocks = torch.nn.functional.pad(x, (0, -k % 32)).view(x.shape[0], -1, 32)
        largest = blocks.abs().amax(dim=-1, keepdim=True).expand_as(blocks).reshape(x.shape[0], -1)[:, :k]
        limit = limit + 2.0 ** -22 * (largest @ w.abs().t())
    return limit + half_ulp(want.abs() + limit, dtype_out)


PRODUCTS = [(1, 1, 1), (1, 32, 7), (3, 33, 130), (8, 1024, 4096), (16, 4096, 640), (17, 2080, 129), (33, 127, 200), (64, 512, 1000),
            (77, 849, 503), (128, 256, 128), (129, 640, 257), (255, 384, 384), (300, 5000, 77), (513, 1184, 640)]


@pytest.mark.parametrize("kind", ["bf16", "f32", "mx4"])
@pytest.mark.parametrize("n,k,m", PRODUCTS)
def test_product_with_weights_in_four_bits(n, k, m, kind):
    from inferrs_b200 import kernels as K
    x = rand((n, k), 3) * torch.exp(rand((n, k), 4))
    w = K.quantize_mx4(0.02 * rand((m, k), 5))
    dense = torch.empty((m, k), device="cuda")
    K.dequantize_mx4(w, dense)
    if kind == "mx4":
        given = K.quantize_mx4(x)
        x = plain.values4(x)[0]
    else:
        given = x.to(DT[kind])
        x = given.double()
    want = x @ dense.double().t()
    for out_type in DT.values():
        out = torch.full((n, m), float("nan"), device="cuda").to(out_type)
        K.linear_mx4(given, w, out)
        limit = product_limit(x, dense.double(), kind, out_type, want)
        assert bool(((out.double() - want).abs() <= limit).all())
        again = torch.empty_like(out)
        K.linear_mx4(given, w, again)
        assert torch.equal(again, out)                 # the same sums every time
    assert K.few_bits_faults() == {}


@pytest.mark.parametrize("kind", ["bf16", "f32", "mx4"])
@pytest.mark.parametrize("n,k,m", [(1, 4096, 300), (8, 2080, 1000), (16, 4096, 520), (30, 3000, 700), (60, 4100, 400)])
def test_product_of_few_rows_cut_every_way(n, k, m, kind):
    """Tiles of every height, K in every number of parts, rings that are shorter and longer than what they carry."""
    from inferrs_b200 import kernels as K
    x, w = rand((n, k), 13).to(DT.get(kind, torch.bfloat16)), K.quantize_mx4(0.02 * rand((m, k), 14))
    dense = torch.empty((m, k), device="cuda")
    K.dequantize_mx4(w, dense)
    given = K.quantize_mx4(x) if kind == "mx4" else x
    x = plain.values4(x)[0] if kind == "mx4" else x.double()
    want = x @ dense.double().t()
    limit = product_limit(x, dense.double(), kind, torch.float32, want)
    for tile_rows, splits in ((128, 1), (128, 2), (128, 4), (128, 8), (88, 1), (88, 8), (64, 2), (40, 4), (24, 1), (8, 1), (8, 8)):
        out = torch.full((n, m), float("nan"), device="cuda")
        K.linear_mx4(given, w, out, tile_rows, splits)
        assert bool(((out.double() - want).abs() <= limit).all()), (tile_rows, splits)
    assert K.few_bits_faults() == {}
    for bad in ((4, 1), (136, 1), (128, 16), (24, 16), (128, -1)):
        with pytest.raises(K.KernelError):
            K.linear_mx4(given, w, out, *bad)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("pad_x,pad_y", [(8, 8), (1, 3)])
def test_product_of_rows_that_lie_apart(pad_x, pad_y, kind):
    from inferrs_b200 import kernels as K
    for n in (5, 40, 200):
        x, w = rand((n, 320), 6).to(DT[kind]), K.quantize_mx4(rand((200, 320), 7))
        plain_out, out = torch.empty((n, 200), dtype=DT[kind], device="cuda"), apart(torch.zeros((n, 200), device="cuda").to(DT[kind]), pad_y)
        K.linear_mx4(x, w, plain_out)
        K.linear_mx4(apart(x, pad_x), w, out)
        assert torch.equal(out, plain_out)


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
def test_a_row_does_not_depend_on_the_others(kind):
    """Rows that hold no numbers reach no other row, and no other feature where a weight is none."""
    from inferrs_b200 import kernels as K
    for n in (4, 20, 150):
        x, dense = rand((n, 256), 8), rand((300, 256), 9)
        clean = torch.empty((n, 300), device="cuda")
        give = (lambda t: t.bfloat16()) if kind == "bf16" else K.quantize_mx4
        K.linear_mx4(give(x), K.quantize_mx4(dense), clean)
        x[1, 7], x[2, 40], dense[5, 9] = float("nan"), float("inf"), float("nan")
        out = torch.empty_like(clean)
        K.linear_mx4(give(x), K.quantize_mx4(dense), out)
        assert not bool(out[1].isfinite().any()) and not bool(out[2].isfinite().any()) and not bool(out[:, 5].isfinite().any())
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1], keep[2], keep[:, 5] = False, False, False
        assert torch.equal(out[keep], clean[keep])


def test_product_of_bfloat16_rows_of_any_size():
    """Numbers of one block far apart, tiny and huge rows, zeros: the pieces keep a row's precision."""
    from inferrs_b200 import kernels as K
    for n in (8, 100):
        x = rand((n, 512), 10)
        x[0] *= 1e30
        x[1] *= 1e-30
        x[2] = 0
        x[3, ::32] *= 1e4
        x[4] = torch.exp2(torch.randint(-14, 1, (512,), generator=gen(1), device="cuda").float())
        x[5, 1::2] = 0
        x = x.bfloat16()
        w = K.quantize_mx4(rand((160, 512), 11))
        dense = torch.empty((160, 512), device="cuda")
        K.dequantize_mx4(w, dense)
        want = x.double() @ dense.double().t()
        out = torch.empty((n, 160), device="cuda")
        K.linear_mx4(x, w, out)
        assert bool(((out.double() - want).abs() <= product_limit(x.double(), dense.double(), "bf16", torch.float32, want)).all())
        assert bool((out[2] == 0).all())


# ---- keys and values in 8 bits ----------------------------------------------------------------------------------------------
def table_for(needed, page, seed, spare=3):
    """A table of pages for requests of ``needed`` tokens, scattered over a pool with ``spare`` pages of nobody."""
    counts = [-(-n // page) for n in needed]
    order = torch.randperm(sum(counts) + spare, generator=gen(seed), device="cuda").int()
    table = torch.full((len(needed), max(counts) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    return table, sum(counts) + spare


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,d,page,rot,interleaved,norm,portions,cached", [
    (4, 2, 128, 16, 128, False, True, (1, 1, 1), 17), (32, 8, 128, 16, 128, False, True, (40, 3), 0),
    (8, 8, 64, 32, 64, False, False, (1,), 0), (5, 1, 64, 16, 32, True, True, (7, 1, 30), 5), (4, 4, 80, 16, 0, False, True, (9,), 100),
    (2, 1, 256, 64, 256, False, False, (70,), 1), (6, 2, 12, 8, 6, False, True, (3, 2), 9), (64, 8, 128, 16, 64, True, True, (33,), 0)])
def test_keys_and_values_join_the_cache_in_eight_bits(heads, kv, d, page, rot, interleaved, norm, portions, cached, dtype):
    from inferrs_b200 import kernels as K
    n, needed = sum(portions), [cached + c for c in portions]
    table, n_pages = table_for(needed, page, 3)
    pages = K.Kv8Pages.zeros(n_pages, kv, page, d, "cuda")
    pages.k.view(torch.uint8).fill_(77)
    pages.v.view(torch.uint8).fill_(77)
    pages.k_scale.fill_(3.0)
    pages.v_scale.fill_(3.0)
    qkv = apart(rand((n, (heads + 2 * kv) * d), 4).to(DT[dtype]), 8)
    weights = [(1 + 0.1 * rand((d,), s)).to(DT[dtype]) if norm else None for s in (5, 6)]
    angle = rand((max(needed) + 1, max(rot // 2, 1)), 7) * 3
    cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
    pos = torch.cat([torch.arange(cached, cached + c) for c in portions]).int().cuda()
    req = torch.cat([torch.full((c,), i) for i, c in enumerate(portions)]).int().cuda()
    q = torch.empty((n, heads, d), dtype=DT[dtype], device="cuda")
    K.qk_norm_rope_store_kv8(qkv, heads, kv, d, weights[0], weights[1], 1e-6, cos, sin, rot, pos, req, table, pages, q,
                             interleaved=interleaved)
    x = qkv.double().reshape(n, heads + 2 * kv, d)
    want_q = plain.turned(x[:, :heads], weights[0], 1e-6, cos, sin, rot, pos, interleaved)
    # norm, rotation and products in float32: a dozen roundings of numbers up to the vector's largest
    slack = 12 * 2.0 ** -24 * 1.5 * want_q.abs().amax(dim=-1, keepdim=True)
    assert bool(((q.double() - want_q).abs() <= slack + half_ulp(want_q.abs() + slack, DT[dtype])).all())
    want_k = plain.turned(x[:, heads:heads + kv], weights[1], 1e-6, cos, sin, rot, pos, interleaved)
    at, place = table[req.long(), (pos // page).long()].long(), (pos % page).long()
    for got, scales, vectors in ((pages.k, pages.k_scale, want_k), (pages.v, pages.v_scale, x[:, heads + kv:])):
        codes, scale = plain.to8(vectors)
        close = scales[at, :, place].double()
        assert bool(((close - scale).abs() <= 30 * 2.0 ** -24 * scale).all())
        mine = got.view(torch.uint8)[at, :, place].view(torch.float8_e4m3fn).double()
        # a code is the nearest to x * 448 / a, which may be off by 2^-19 of 448 before it is rounded
        exact = vectors / scale.unsqueeze(-1)
        step = torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=2.0 ** -6))) - 3)
        assert bool(((mine - exact).abs() <= step / 2 + 448 * 2.0 ** -18).all())
        assert float((mine == codes).double().mean()) > 0.999 or mine.numel() < 4000
    untouched = torch.ones((n_pages, page), dtype=torch.bool, device="cuda")
    untouched[at, place] = False
    untouched = untouched[:, None].expand(n_pages, kv, page)
    for t, fill in ((pages.k.view(torch.uint8), 77), (pages.v.view(torch.uint8), 77), (pages.k_scale, 3.0), (pages.v_scale, 3.0)):
        assert bool((t[untouched] == fill).all())
    assert K.few_bits_faults() == {}


def test_vectors_of_zeros_tiny_numbers_and_none():
    from inferrs_b200 import kernels as K
    x = torch.zeros((5, 3, 64), device="cuda")
    x[0], x[1], x[2] = 1e-33, 1e-29, 1.0
    x[3, 1:, 5], x[4, 1:, 6] = float("inf"), float("nan")
    pages = K.Kv8Pages.zeros(2, 1, 16, 64, "cuda")
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    pos, req = torch.arange(5, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    q = torch.empty((5, 1, 64), device="cuda")
    K.qk_norm_rope_store_kv8(x.view(5, 192), 1, 1, 64, None, None, 0.0, None, None, 0, pos, req, table, pages, q)
    for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        back = codes.float()[0, 0] * scale[0, 0].unsqueeze(-1)
        assert bool((back[0] == 0).all()) and float(scale[0, 0, 0]) == 0
        assert torch.allclose(back[1], torch.full((64,), 1e-29, device="cuda"), rtol=1e-6)
        assert torch.allclose(back[2], torch.ones(64, device="cuda"), rtol=1e-6)
        assert not bool(back[3].isfinite().any()) and not bool(back[4].isfinite().any())


def test_rows_without_a_place_in_the_cache():
    """A row outside the rotation tables is left out and reported; one without a page writes its query only."""
    from inferrs_b200 import kernels as K
    K.few_bits_faults()
    qkv = rand((4, 3 * 64), 1)
    pages = K.Kv8Pages.zeros(2, 1, 16, 64, "cuda")
    table = torch.tensor([[1], [-1], [9]], dtype=torch.int32, device="cuda")
    cos = torch.ones((8, 32), device="cuda")
    q = torch.full((4, 1, 64), 7.0, device="cuda")
    pos = torch.tensor([3, 8, 2, 1], dtype=torch.int32, device="cuda")
    req = torch.tensor([0, 0, 1, 2], dtype=torch.int32, device="cuda")
    K.qk_norm_rope_store_kv8(qkv, 1, 1, 64, None, None, 0.0, cos, torch.zeros_like(cos), 64, pos, req, table, pages, q)
    assert K.few_bits_faults() == {K.FEW_BITS_WORDS[0]: 2}
    assert K.few_bits_faults() == {}
    assert torch.equal(q[[0, 2, 3], 0], qkv[[0, 2, 3], :64]) and bool((q[1] == 7).all())
    written = pages.k_scale[1, 0].nonzero().flatten().tolist()
    assert written == [3] and not bool(pages.k_scale[0].any())


# ---- attention over 8-bit keys and values ------------------------------------------------------------------------------------
def filled(lengths, kv, d, page, seed):
    from inferrs_b200 import kernels as K
    table, n_pages = table_for([max(1, n) for n in lengths], page, seed)
    pages = K.Kv8Pages.zeros(n_pages, kv, page, d, "cuda")
    for name, t, s in (("k", pages.k, pages.k_scale), ("v", pages.v, pages.v_scale)):
        x = rand(t.shape, seed + len(name + "k") + (name == "v"))
        a = x.abs().amax(-1)
        t.copy_((x * (448 / a).unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn))
        s.copy_(a / 448 * torch.exp(0.5 * rand(a.shape, seed + 9)))
    # what no request has written holds no numbers
    mine = torch.zeros((n_pages, page), dtype=torch.bool, device="cuda")
    for i, n in enumerate(lengths):
        j = torch.arange(n, device="cuda")
        mine[table[i].long()[j // page], j % page] = True
    foreign = ~mine[:, None].expand(n_pages, kv, page)
    for t, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        t.view(torch.uint8)[foreign] = 0x7F
        s[foreign] = float("nan")
    return pages, table


def attention_limit(want, weight, size, d, longest, dtype):
    """Scores: d products in float32 and as many additions (2^-23 of their sum), 2^-22 of the score itself for its way to the
    exponent and 2^-21 for the exponential; a probability is rounded to 11 bits in the bfloat16 form; sums of up to
    ``longest`` of them; the result's rounding."""
    off = 2 * size * (d + 12) * 2.0 ** -23 + 2.0 ** -20 + (longest + 64) * 2.0 ** -24
    if dtype == torch.bfloat16:
        off = off + 2.0 ** -10
    limit = off * weight
    return limit + half_ulp(want.abs() + limit, dtype)


def check_attention(lengths, heads, kv, d, page, span, dtype, seed=1, spread=1.0, scale=None):
    from inferrs_b200 import kernels as K
    pages, table = filled(lengths, kv, d, page, seed)
    n = len(lengths)
    q = (spread * rand((n, heads, d), seed + 20)).to(dtype)
    pos = torch.tensor([length - 1 for length in lengths], dtype=torch.int32, device="cuda")
    req = torch.arange(n, dtype=torch.int32, device="cuda")
    out = apart(torch.full((n, heads * d), float("nan"), device="cuda").to(dtype), 8)
    scale = d ** -0.5 if scale is None else scale
    longest = max(max(lengths), 1)
    K.paged_attention_kv8(q, pages, table, req, pos, scale, span or None, out, longest)
    codes = [t.double() for t in (pages.k, pages.v)]
    scales = [s.double() for s in (pages.k_scale, pages.v_scale)]
    want, weight, size = plain.attention(q, codes[0], codes[1], scales[0], scales[1], table, req, pos, scale, span)
    got = out.double().view(n, heads, d)
    assert bool(got.isfinite().all())
    assert bool(((got - want).abs() <= attention_limit(want, weight, size, d, longest, dtype)).all())
    again = torch.empty_like(out)
    K.paged_attention_kv8(q, pages, table, req, pos, scale, span or None, again, longest)
    assert torch.equal(out, again)                      # the same sums every time
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,d,page", [(16, 8, 128, 16), (32, 8, 128, 16), (20, 4, 64, 32), (32, 2, 128, 64), (4, 4, 64, 16),
                                             (7, 1, 128, 8), (6, 2, 80, 16), (2, 1, 256, 16), (24, 1, 64, 16), (3, 3, 12, 4)])
def test_attention_over_eight_bit_pages(heads, kv, d, page, dtype):
    check_attention([1, 2, 15, 16, 17, 33, 64, 65, 127, 300, 1025], heads, kv, d, page, 0, DT[dtype])


@pytest.mark.parametrize("span", [1, 2, 16, 50, 100, 1000, -32, -7])
def test_attention_over_eight_bit_pages_with_a_window(span):
    for dtype in DT.values():
        check_attention([1, 16, 31, 100, 101, 777], 8, 2, 128, 16, span, dtype, seed=3)


@pytest.mark.parametrize("lengths", [(5000,), (4097, 1), (2000, 1, 0, 700, 64), (300,) * 150, tuple(range(1, 60, 3)), (9000, 8999, 8998)])
def test_attention_over_eight_bit_pages_cut_many_ways(lengths):
    """Long contexts are cut and joined; a request of no keys among others (position -1) gets zeros."""
    got = check_attention(list(lengths), 8, 2, 128, 16, 0, torch.bfloat16, seed=5)
    for i, n in enumerate(lengths):
        if n == 0:
            assert bool((got[i] == 0).all())
    check_attention(list(lengths)[:4], 8, 2, 64, 16, 0, torch.bfloat16, seed=6)


def test_attention_over_eight_bit_pages_with_sharp_and_flat_scores():
    """Scores of hundreds (one key takes all), of nothing (an even mean), queries of zeros and of great size."""
    check_attention([40, 3000], 8, 2, 128, 16, 0, torch.bfloat16, seed=7, spread=60.0)
    check_attention([40, 3000], 8, 2, 128, 16, 0, torch.bfloat16, seed=7, spread=0.0)
    check_attention([40, 3000], 8, 2, 128, 16, 0, torch.bfloat16, seed=7, spread=1e-20, scale=1e18)
    check_attention([40, 3000], 8, 2, 128, 16, 0, torch.bfloat16, seed=7, spread=1e15, scale=1e-17)


def test_attention_over_eight_bit_pages_whose_scales_are_far_apart():
    """Values a million times smaller than a neighbour's keep their precision where the neighbour is not looked at."""
    from inferrs_b200 import kernels as K
    pages, table = filled([200], 1, 128, 16, 8)
    far = table[0].long()[torch.tensor([3, 7])]
    pages.v_scale[far[0], :, 2] *= 1e9
    pages.v_scale[far[1], :, 5] *= 1e-9
    keys = pages.k.double() * pages.k_scale.double().unsqueeze(-1)
    loud = keys[far[0], 0, 2]
    q = (-8 * loud / loud.norm()).float().bfloat16().view(1, 1, 128).repeat(1, 4, 1)
    q[0, 1] = -q[0, 0]
    pos, req = torch.tensor([199], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty((1, 512), dtype=torch.bfloat16, device="cuda")
    K.paged_attention_kv8(q, pages, table, req, pos, 3.0, None, out, 200)
    want, weight, size = plain.attention(q, pages.k.double(), pages.v.double(), pages.k_scale.double(), pages.v_scale.double(),
                                         table, req, pos, 3.0, 0)
    limit = attention_limit(want, weight, size, 128, 200, torch.bfloat16)
    assert bool(((out.double().view(1, 4, 128) - want).abs() <= limit).all())


# ---- refusals ------------------------------------------------------------------------------------------------------------
def test_refusals():
    from inferrs_b200 import kernels as K
    x = rand((4, 64), 1)
    w = K.quantize_mx4(x)
    out = torch.empty((4, 4), device="cuda")
    bad = [lambda: K.quantize_mx4(x.cpu()), lambda: K.quantize_mx4(x.half()), lambda: K.quantize_mx4(x.t()), lambda: K.quantize_mx4(x[0]),
           lambda: K.quantize_mx4(x, K.Mx4Matrix.empty(5, 64, "cuda")), lambda: K.Mx4Matrix.empty(3, 0, "cuda"),
           lambda: K.Mx4Matrix(w.codes, w.scales, 5, 64), lambda: K.Mx4Matrix(w.codes, w.scales[:, :1], 4, 64),
           lambda: K.Mx4Matrix(w.codes.cpu(), w.scales, 4, 64), lambda: K.Mx4Matrix(w.codes.int(), w.scales, 4, 64),
           lambda: K.dequantize_mx4(w, torch.empty((4, 65), device="cuda")), lambda: K.dequantize_mx4(w, torch.empty((4, 64))),
           lambda: K.linear_mx4(x[:, :32], w, out), lambda: K.linear_mx4(x, w, out[:3]), lambda: K.linear_mx4(x.half(), w, out),
           lambda: K.linear_mx4(x, w, out.t()[:, :3]), lambda: K.linear_mx4(x, w, out.int())]
    pages = K.Kv8Pages.zeros(2, 1, 16, 64, "cuda")
    table, one = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    qkv, q = rand((1, 192), 2), torch.empty((1, 1, 64), device="cuda")
    cos = torch.ones((4, 32), device="cuda")

    def store(**kw):
        a = dict(qkv=qkv, n_heads=1, n_kv_heads=1, head_dim=64, q_weight=None, k_weight=None, eps=0.0, cos=cos, sin=cos, rot_dim=64,
                 positions=one, row_request=one, block_table=table, pages=pages, q_out=q)
        a.update(kw)
        return lambda: K.qk_norm_rope_store_kv8(**a)

    def attend(**kw):
        a = dict(q=q, pages=pages, block_table=table, row_request=one, positions=one, scale=1.0, window=None,
                 out=torch.empty((1, 64), device="cuda"), max_kv_len=1)
        a.update(kw)
        return lambda: K.paged_attention_kv8(**a)

    bad += [store(qkv=qkv[:, :128]), store(qkv=qkv.bfloat16()), store(q_out=q.half()), store(n_heads=2), store(head_dim=32),
            store(q_weight=torch.ones(32, device="cuda")), store(rot_dim=63), store(rot_dim=32), store(sin=cos[:2]),
            store(positions=one.long()), store(positions=torch.zeros(2, dtype=torch.int32, device="cuda")), store(block_table=table[0]),
            store(q_weight=torch.ones(64, device="cuda"), k_weight=torch.ones(64, device="cuda").bfloat16()),
            attend(q=q.bfloat16()), attend(q=q[0]), attend(out=torch.empty((1, 65), device="cuda")), attend(positions=one.long()),
            attend(row_request=torch.zeros(2, dtype=torch.int32, device="cuda")), attend(block_table=table.long()),
            lambda: K.Kv8Pages(pages.k, pages.v, pages.k_scale, pages.v_scale[:1]),
            lambda: K.Kv8Pages(pages.k.view(torch.uint8), pages.v, pages.k_scale, pages.v_scale),
            lambda: K.Kv8Pages.zeros(1, 1, 16, 6, "cuda")]
    for i, call in enumerate(bad):
        with pytest.raises(K.KernelError):
            call()
            pytest.fail(f"call {i} was taken")
    attend()()
    store()()


def test_on_a_stream_of_its_own_and_in_a_captured_graph():
    """The operators launch on the current stream and allocate nothing that a replay would miss."""
    from inferrs_b200 import kernels as K
    x, w = rand((8, 512), 1).bfloat16(), K.quantize_mx4(rand((300, 512), 2))
    pages, table = filled([700], 2, 128, 16, 4)
    q = rand((1, 4, 128), 5).bfloat16()
    pos, req = torch.tensor([699], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    y, y4, out = (torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((8, 300), (8, 300), (1, 512)))

    def step():
        K.linear_mx4(x, w, y)
        K.linear_mx4(K.quantize_mx4(x), w, y4)
        K.paged_attention_kv8(q, pages, table, req, pos, 0.1, None, out, 700)

    step()
    want = [t.clone() for t in (y, y4, out)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in (y, y4, out):
            t.zero_()
        step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (y, y4, out)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        for t in (y, y4, out):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (y, y4, out)))


@pytest.mark.parametrize("heads,kv,d,span", [(8, 2, 128, 0), (32, 8, 128, 20), (16, 16, 64, 0), (20, 4, 64, -16), (2, 1, 256, 0), (5, 1, 128, 7)])
def test_attention_of_prompts_over_eight_bit_pages(heads, kv, d, span):
    """Tiles of a prompt's tokens, some short, some places of the list without a tile, beside rows one by one."""
    from inferrs_b200 import kernels as K
    portions, cached = (37, 1, 12), (100, 5, 0)
    lengths = [c + p for c, p in zip(cached, portions)]
    pages, table = filled(lengths, kv, d, 16, 2)
    n = sum(portions)
    q = rand((n, heads, d), 3).bfloat16()
    pos = torch.cat([torch.arange(c, c + p) for c, p in zip(cached, portions)]).int().cuda()
    req = torch.cat([torch.full((p,), i) for i, p in enumerate(portions)]).int().cuda()
    starts = [0, 37, 38, 50]
    tokens = K.kv8_tile_tokens(heads, kv, d)
    tile_list = [(i, r) for i in range(3) for r in range(starts[i], starts[i + 1], tokens)]
    tile_list.insert(1, (-1, 0))
    tile_req, tile_row0 = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in zip(*tile_list))
    q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out, one = (torch.full((n, heads * d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scale = d ** -0.5
    K.paged_attention_kv8(q, pages, table, req, pos, scale, span, out, max(lengths), tiles=(tile_req, tile_row0, len(tile_list), q_start, tokens))
    K.paged_attention_kv8(q, pages, table, req, pos, scale, span, one, max(lengths))
    want, weight, size = plain.attention(q, pages.k.double(), pages.v.double(), pages.k_scale.double(), pages.v_scale.double(),
                                         table, req, pos, scale, span)
    limit = attention_limit(want, weight, size, d, max(lengths), torch.bfloat16)
    for got in (out, one):
        assert bool(((got.double().view(n, heads, d) - want).abs() <= limit).all())


# ---- rows that start anywhere in memory ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,offset", [(1, 0), (2, 0), (3, 1), (4, 0), (4, 2), (6, 1), (8, 0), (8, 1), (8, 4), (12, 4)])
def test_rows_that_start_anywhere(pad, offset, dtype):
    """The same bits as rows side by side give, nothing written beside the rows."""
    from inferrs_b200 import kernels as K
    width = 271
    whole = rand((37, width + pad + offset), 5).to(DT[dtype])
    x = whole[:, offset:offset + width]
    w, same = K.quantize_mx4(x), K.quantize_mx4(x.contiguous())
    assert torch.equal(w.codes, same.codes)
    room = torch.full_like(whole, 7.0)
    straight = torch.empty((37, width), dtype=DT[dtype], device="cuda")
    K.dequantize_mx4(w, room[:, offset:offset + width])
    K.dequantize_mx4(same, straight)          # (scales behind the last row are not written: what counts are the values)
    assert torch.equal(room[:, offset:offset + width], straight)
    assert bool((room[:, :offset] == 7).all()) and bool((room[:, offset + width:] == 7).all())
    m = K.quantize_mx4(rand((130, width), 6))
    for rows in (1, 7, 37):
        got, want = (torch.empty((rows, 130), device="cuda") for _ in range(2))
        K.linear_mx4(x[:rows], m, got)
        K.linear_mx4(x[:rows].contiguous(), m, want)
        assert torch.equal(got, want)


@pytest.mark.parametrize("d,weights", [(64, "bf16"), (128, "bf16"), (128, "f32"), (256, "bf16")])
def test_keys_take_the_nearest_codes(d, weights):
    """Of keys that the kernel for whole heads turns, every code is the one that 64-bit arithmetic gives (a key of zeros beside them stays one)."""
    from inferrs_b200 import kernels as K
    n, heads, kv = 700, 3, 5
    table, n_pages = table_for([n], 16, 1)
    pages = K.Kv8Pages.zeros(n_pages, kv, 16, d, "cuda")
    qkv = rand((n, (heads + 2 * kv) * d), 4).bfloat16()
    qkv[5, heads * d:(heads + 2) * d] = 0
    q_weight, k_weight = ((1 + 0.1 * rand((d,), s)).to(DT[weights]) for s in (5, 6))
    angle = rand((n, d // 2), 7) * 3
    pos, req = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    q = torch.empty((n, heads, d), dtype=torch.bfloat16, device="cuda")
    K.qk_norm_rope_store_kv8(qkv, heads, kv, d, q_weight, k_weight, 1e-6, angle.cos(), angle.sin(), d, pos, req, table, pages, q)
    want = plain.turned(qkv.double().reshape(n, heads + 2 * kv, d)[:, heads:heads + kv], k_weight, 1e-6, angle.cos(), angle.sin(), d, pos, False)
    codes, _ = plain.to8(want)
    got = pages.k.view(torch.uint8)[table[0].long()[(pos // 16).long()], :, (pos % 16).long()].view(torch.float8_e4m3fn).double()
    wrong = int((got != codes).sum())
    assert wrong == 0 if weights == "bf16" else wrong < 3      # (float32 weights: a product of 48 bits is rounded to 24)
    assert bool((got[5, :2] == 0).all())


@pytest.mark.parametrize("kind", ["bf16", "f32", "mx4"])
@pytest.mark.parametrize("n,k,m", [(2100, 300, 9000), (700, 4100, 8200), (50, 260, 8200), (33, 129, 8300), (64, 2080, 8448), (97, 64, 20000), (4000, 1, 513),
                                   (193, 768, 256), (200, 2000, 127)])
def test_products_of_many_tiles(n, k, m, kind):
    """More tiles than pairs of CTAs, so that pairs take several and accumulators take turns; K of fewer stages than there is room for; a pair's
    second half, or most of it, behind the last row of W."""
    from inferrs_b200 import kernels as K
    x = rand((n, k), 13)
    w = K.quantize_mx4(0.02 * rand((m, k), 15))
    dense = torch.empty((m, k), device="cuda")
    K.dequantize_mx4(w, dense)
    given = K.quantize_mx4(x) if kind == "mx4" else x.to(DT[kind])
    x = plain.values4(x)[0].double() if kind == "mx4" else given.double()
    want = x @ dense.double().t()
    for out_type, pad in ((torch.bfloat16, 0), (torch.float32, 3)):
        room = torch.full((n, m + pad), 7.0, device="cuda").to(out_type)
        out = room[:, :m]
        K.linear_mx4(given, w, out)
        limit = product_limit(x, dense.double(), kind, out_type, want)
        assert bool(((out.double() - want).abs() <= limit).all())
        assert bool((room[:, m:] == 7).all())
    assert K.few_bits_faults() == {}
