"""Attention of drafted tokens, kept tokens, copied pages and log probabilities against their definitions in 64 bits."""
from __future__ import annotations

import random

import pytest
import torch

import plain_drafts as plain
from inferrs_b200 import kernels
from inferrs_b200.engine.batch import tree_masks

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert kernels.attention_tree_error() == 0 and kernels.log_probs_error() == 0


# ---- attention ---------------------------------------------------------------------------------------------------------
def drafted(seed, contexts, trees, heads, kv, d, page, dtype, chain=False, spare=0, words=None):
    """Everything that a call takes, with pages in no order, leftovers in the places that hold no key, and rows behind the last."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    parents = [[(i - 1 if chain else rng.randrange(max(-1, i - 6), i)) for i in range(t)] for t in trees]
    masks, depths = tree_masks(parents, words)
    starts = [sum(trees[:i]) for i in range(len(trees) + 1)]
    counts = [max(1, -(-(c + t) // page)) for c, t in zip(contexts, trees)]
    order = torch.randperm(sum(counts) + 2, generator=g).tolist()
    table = torch.full((len(trees), max(counts)), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    make = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    n = starts[-1]
    k, v = make(sum(counts) + 2, kv, page, d).to(dtype), make(sum(counts) + 2, kv, page, d).to(dtype)
    used = torch.zeros((sum(counts) + 2, page), dtype=torch.bool)
    for r in range(len(trees)):
        for j in range(contexts[r] + trees[r]):
            used[table[r, j // page], j % page] = True
    k[~used[:, None].expand(-1, kv, -1)] = float("nan")
    v[~used[:, None].expand(-1, kv, -1)] = float("inf")
    positions = [contexts[r] + int(depths[starts[r] + i]) for r in range(len(trees)) for i in range(trees[r])] + [0] * spare
    return dict(q=(2 * make(n + spare, heads, d)).to(dtype).to(DEV), k=k.to(DEV), v=v.to(DEV), table=table.to(DEV), q_start=ints(starts),
                context=ints(contexts), positions=ints(positions), seen=ints(masks.tolist() + [[0] * masks.shape[1]] * spare),
                most=max(trees), longest=max(c + t for c, t in zip(contexts, trees)))


def attend(c, span=None, out=None, scale=None, positions=True):
    n, h, d = c["q"].shape
    if out is None:
        out = torch.full((n, h * d), 7.0, dtype=c["q"].dtype, device=DEV)
    kernels.paged_attention_tree(c["q"], c["k"], c["v"], c["table"], c["q_start"], c["context"], c["positions"] if positions else None,
                                 c["seen"], scale or d ** -0.5, span, out, c["most"], c["longest"])
    return out


def check(c, out, span=0, scale=None):
    n, h, d = c["q"].shape
    want, off = plain.tree_attention(c["q"], c["k"], c["v"], c["table"], c["q_start"], c["context"], c["positions"], c["seen"],
                                     scale or d ** -0.5, span or 0)
    last = int(c["q_start"][-1])
    got = out.cpu().double().view(n, h, d)
    assert (got[last:] == 7.0).all()
    got, want, off = got[:last], want[:last], off[:last]
    some = torch.isfinite(want)
    assert (torch.isfinite(got) == some).all()
    bound = off + plain.HALF[out.dtype] * (want.abs() + off) + 1e-30
    assert ((got - want).abs() <= bound)[some].all(), ((got - want).abs() / bound)[some].max()


SHAPES = [
    # contexts, trees, heads, kv, d, page, dtype
    ([300], [8], 16, 8, 128, 16, BF),
    ([0], [1], 4, 4, 128, 16, BF),
    ([1], [1], 8, 1, 64, 16, BF),
    ([127, 128, 129], [1, 2, 3], 8, 2, 128, 16, BF),
    ([0, 5, 0], [40, 33, 1], 8, 2, 128, 16, BF),
    ([255, 0, 700], [16, 16, 9], 32, 8, 128, 32, BF),
    ([513, 90], [64, 64], 16, 4, 128, 16, BF),
    ([400], [100], 20, 4, 128, 64, BF),
    ([37, 500], [130, 7], 8, 1, 128, 16, BF),
    ([1500], [5], 10, 2, 64, 16, BF),
    ([600, 3], [70, 70], 14, 2, 64, 8, BF),
    ([200, 81], [12, 31], 6, 3, 80, 16, BF),
    ([90], [9], 4, 2, 20, 4, BF),
    ([50], [9], 4, 2, 33, 7, BF),
    ([140], [11], 4, 2, 256, 16, BF),
    ([130, 64], [11, 5], 8, 2, 128, 48, BF),
    ([130, 300], [11, 5], 8, 2, 128, 4, BF),
    ([500, 300, 7], [11, 80, 3], 8, 2, 128, 256, BF),
    ([500, 129], [11, 70], 8, 2, 64, 128, BF),
    ([300, 77], [13, 8], 16, 8, 128, 16, F32),
    ([0, 31, 32, 33], [1, 2, 3, 64], 4, 2, 64, 16, F32),
    ([45], [20], 6, 2, 36, 5, F32),
    ([45], [20], 6, 2, 7, 5, F32),
    ([60], [3], 2, 1, 512, 16, F32),
    ([900], [33], 12, 4, 128, 64, F32),
]


@pytest.mark.parametrize("case", range(len(SHAPES)))
@pytest.mark.parametrize("span", [None, 50, -64])
def test_tree_attention(case, span):
    contexts, trees, heads, kv, d, page, dtype = SHAPES[case]
    c = drafted(case, contexts, trees, heads, kv, d, page, dtype, chain=case % 3 == 0, spare=3 if case % 2 else 0)
    check(c, attend(c, span), span)


@pytest.mark.parametrize("d,heads,kv,most,span", [(128, 16, 8, 9, None), (64, 16, 8, 20, None), (128, 8, 8, 40, 6200), (128, 16, 8, 70, None),
                                                  (64, 32, 8, 64, None), (128, 32, 8, 100, None)])
def test_tree_attention_requests_of_very_different_length(d, heads, kv, most, span):
    """More CTAs than run at once: the long requests' keys go in slices that are joined by a kernel of their own."""
    rng = random.Random(most)
    contexts = [0, 3300, 5, 6500, 130, 64, 7, 2000, 33, 1]
    trees = [rng.randrange(1, most + 1) for _ in contexts]
    trees[3], trees[4], trees[5] = most, 0, 1
    c = drafted(21, contexts, trees, heads, kv, d, 16, BF, spare=2)
    assert c["longest"] > kernels.TREE_SLICE and 2 * len(contexts) * kv > 148
    out = attend(c, span)
    check(c, out, span)
    c["v"][c["table"][3, 6500 // 16], :, 6500 % 16] = float("nan")      # the first drafted token of the longest one
    got = attend(c, span).float().view(out.shape[0], heads, d)
    start = int(c["q_start"][3])
    hit = torch.zeros(out.shape[0], dtype=torch.bool, device=DEV)
    hit[start:start + most] = (c["seen"][start:start + most, 0] & 1).bool()
    assert torch.isnan(got[hit]).all() and torch.isfinite(got[~hit]).all()


@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (128, 24), (64, 256)])
@pytest.mark.parametrize("requests,span", [(5, None), (5, 900), (5, -700), (10, None), (10, 64)])
def test_tree_attention_many_rows_over_many_keys(d, page, requests, span):
    """Enough CTAs that two sets of rows share their keys: in clusters (5 requests) and alone (10)."""
    contexts, trees = ([1100, 900, 0, 1000, 130], [40, 37, 33, 40, 1])
    if requests == 10:
        contexts, trees = contexts[1:] + [300, 5, 128, 127, 400, 64], trees[1:] + [40, 39, 2, 0, 36, 40]
    c = drafted(31, contexts, trees, 32, 8, d, page, BF, chain=page == 24, spare=1)
    out = attend(c, span)
    check(c, out, span)
    # a value that is no number: the rows that see it, no others
    c["v"][c["table"][0, contexts[0] // page], :, contexts[0] % page] = float("nan")
    c["v"][c["table"][1, 3 // page], :, 3 % page] = float("inf")
    got = attend(c, span)
    finite = torch.isfinite(got.float().view(got.shape[0], 32, d)).all(2).all(1)
    hit = torch.zeros(out.shape[0], dtype=torch.bool, device=DEV)
    hit[:trees[0]] = (c["seen"][:trees[0], 0] & 1).bool()
    rows = slice(trees[0], trees[0] + trees[1])
    at = c["positions"][rows]
    if contexts[1] <= 3:                  # (place 3 is a drafted token)
        hit[rows] = (c["seen"][rows, 0] >> (3 - contexts[1]) & 1).bool()
    else:
        hit[rows] = True if span is None else at - span < 3 if span > 0 else at // -span == 0
    assert torch.equal(finite, ~hit)
    assert torch.equal(got[~hit], out[~hit])
    c["table"][0, 2] = -1                 # a page that is not there
    c["v"][c["table"][0, contexts[0] // page], :, contexts[0] % page] = 1.0
    c["v"][c["table"][1, 3 // page], :, 3 % page] = 1.0
    check(c, attend(c, span), span)


def test_tree_attention_many_requests_and_splits():
    rng = random.Random(3)
    contexts = [rng.choice([0, 1, 17, 200, 900]) for _ in range(40)]
    trees = [rng.choice([0, 1, 4, 12]) for _ in range(40)]
    c = drafted(11, contexts, trees, 8, 4, 128, 16, BF)
    check(c, attend(c))
    c = drafted(12, [3000], [7], 8, 1, 128, 16, BF)
    check(c, attend(c))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 64), (BF, 96), (F32, 128)])
def test_tree_attention_any_mask(dtype, d):
    """Masks that no tree has: rows that see nothing of it, not themselves, later ones, bits behind the last token; more words than needed."""
    c = drafted(5, [0, 200, 0], [37, 37, 5], 4, 2, d, 16, dtype, words=4)
    g = torch.Generator().manual_seed(1)
    seen = torch.randint(-2 ** 31, 2 ** 31, c["seen"].shape, generator=g, dtype=torch.int64).to(torch.int32)
    seen[3] = 0
    seen[40] = 0
    seen[-1] = 0
    c["seen"] = seen.to(DEV)
    out = attend(c)
    check(c, out)
    assert (out[3] == 0).all() and (out[-1] == 0).all()
    one = drafted(6, [150, 60], [9, 40], 4, 2, d, 16, dtype)        # fewer words than tokens: the others are not seen
    one["seen"] = one["seen"][:, :1].contiguous()
    check(one, attend(one))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 64), (BF, 48), (F32, 128)])
def test_tree_attention_a_window_that_leaves_nothing(dtype, d):
    """Positions far behind the context: a window sees no key of it; masks without a bit: the row is zeros."""
    c = drafted(7, [300, 40], [6, 3], 4, 2, d, 16, dtype)
    c["positions"] = c["positions"] + 1000
    check(c, attend(c, 64), 64)
    c["seen"] = torch.zeros_like(c["seen"])
    assert (attend(c, 64) == 0).all()


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 64), (BF, 72), (F32, 128)])
def test_tree_attention_what_is_not_seen_does_not_reach_a_row(dtype, d):
    """Infinities and no numbers in keys and values of another branch and ahead of the window; rows that see them have no numbers."""
    c = drafted(8, [260, 10], [24, 6], 4, 2, d, 16, dtype)
    page = c["k"].shape[2]

    def put(pages, r, j, value):
        pages[c["table"][r, j // page], :, j % page, 3] = value

    put(c["k"], 0, 260 + 7, float("nan"))
    put(c["v"], 0, 260 + 9, float("inf"))
    put(c["v"], 0, 260 + 11, float("nan"))
    put(c["k"], 0, 3, float("inf"))
    put(c["v"], 0, 5, float("nan"))
    put(c["v"], 0, 150, float("-inf"))
    out = attend(c, 100)
    n, h = c["q"].shape[:2]
    seen = [[bool(w[j // 32] >> (j % 32) & 1) for j in range(24)] for w in c["seen"][:24].tolist()]
    got = out.view(n, h, d).float().cpu()
    for i in range(24):
        reach = int(c["positions"][i]) - 99
        hit = seen[i][7] or seen[i][9] or seen[i][11] or reach <= 150
        column = got[i, :, 3]
        assert torch.isfinite(column).all() != hit or not hit, (i, hit)
        assert torch.isfinite(column).any().item() != hit, (i, hit)
        if not seen[i][7]:
            assert torch.isfinite(torch.cat((got[i, :, :3], got[i, :, 4:]), 1)).all(), i
    assert torch.isfinite(got[24:]).all()


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 64), (BF, 72), (F32, 128)])
def test_tree_attention_pages_that_are_not_there(dtype, d):
    c = drafted(9, [300, 200], [10, 12], 8, 2, d, 16, dtype)
    c["table"][0, 2] = -1
    c["table"][0, 7] = c["k"].shape[0]
    c["table"][1, 12] = -1        # of drafted tokens and the context's end
    check(c, attend(c))
    c["table"][:] = -1
    assert (attend(c) == 0).all()
    c["table"] = c["table"][:, :0].contiguous()
    assert (attend(c) == 0).all()


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F32, 64)])
def test_tree_attention_rows_that_lie_apart_and_other_scales(dtype, d):
    c = drafted(10, [77, 130], [5, 18], 4, 2, d, 16, dtype)
    n, h = c["q"].shape[:2]
    wide = torch.full((n, h * d + 6), 7.0, dtype=dtype, device=DEV)
    attend(c, out=wide[:, 1:1 + h * d])
    check(c, wide[:, 1:1 + h * d].contiguous())
    assert (wide[:, 0] == 7).all() and (wide[:, 1 + h * d:] == 7).all()
    for scale in (0.5, -0.1, 1e-6):
        check(c, attend(c, scale=scale), scale=scale)
    assert (attend(c, positions=False) == attend(c)).all()


def moved(t, by):
    """The same numbers in memory that starts ``by`` of them off a boundary."""
    flat = torch.empty((t.numel() + by,), dtype=t.dtype, device=DEV)
    flat[by:].copy_(t.flatten())
    return flat[by:].view(t.shape)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 64), (BF, 80), (F32, 128), (F32, 20)])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_tree_attention_tensors_that_start_anywhere(dtype, d, which):
    c = drafted(15, [150, 7], [9, 12], 4, 2, d, 16, dtype)
    for by in (1, 4):
        c[which] = moved(c[which], by)
        check(c, attend(c))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 96), (F32, 64)])
def test_tree_attention_a_cache_without_pages_and_calls_without_rows(dtype, d):
    c = drafted(16, [50, 7], [3, 4], 4, 2, d, 16, dtype)
    empty = dict(c, k=c["k"][:0], v=c["v"][:0])
    assert (attend(empty) == 0).all()
    none = dict(c, q=c["q"][:0].contiguous(), q_start=ints([0, 0, 0]), positions=c["positions"][:0], seen=c["seen"][:0])
    assert attend(none).shape[0] == 0
    lying = dict(c, q_start=ints([-5, 3, 2 ** 31 - 1]), context=ints([-3, 2 ** 31 - 1]))     # read as far as there is anything
    attend(lying)


def test_what_the_calls_refuse():
    c = drafted(17, [50, 7], [3, 4], 4, 2, 64, 16, BF)
    for name, bad in (("q", c["q"].float()), ("q", c["q"].transpose(0, 1)), ("k", c["k"][..., :32]), ("v", c["v"][:3]), ("table", c["table"].long()),
                      ("table", c["table"][:1]), ("q_start", c["q_start"][:2]), ("context", c["context"].float()), ("seen", c["seen"][:2]),
                      ("seen", c["seen"].cpu()), ("context", c["context"].cpu()), ("positions", c["positions"][:1])):
        with pytest.raises(kernels.KernelError):
            attend(dict(c, **{name: bad}), out=torch.zeros((7, 256), dtype=BF, device=DEV))
    with pytest.raises(kernels.KernelError):
        attend(c, span=9, positions=False)
    with pytest.raises(kernels.KernelError):
        attend(c, out=torch.zeros((7, 128), dtype=BF, device=DEV))
    wide = drafted(18, [5], [3], 2, 1, 520, 16, F32)
    with pytest.raises(kernels.KernelError):
        attend(wide)
    pages = torch.zeros((2, 5, 2, 16, 8), device=DEV)
    for args in ((pages, 5, ints([0]), ints([1])), (pages, 1, ints([0]), ints([1, 2])), (pages, 1, ints([0]).long(), ints([1])),
                 (pages[:, ::2], 1, ints([0]), ints([1])), (pages, 1, ints([0]).cpu(), ints([1]))):
        with pytest.raises(kernels.KernelError):
            kernels.copy_pages(*args)
    t, n = ints([[0, 1]]), ints([1])
    for args in ((pages, 3, t, n, t, n), (pages, 1, t, n, ints([[0], [1]]), n), (pages, 1, t, ints([1, 2]), t, n), (pages, 1, t.long(), n, t, n)):
        with pytest.raises(kernels.KernelError):
            kernels.keep_tokens(*args)
    x, one = torch.zeros((3, 50), device=DEV), torch.zeros((3, 1), device=DEV)
    k33 = (ints([[0] * 33] * 3), torch.zeros((3, 33), device=DEV))
    for args in ((x.half(), ints([[1]] * 3), one), (x, ints([[1]] * 2), one), (x, ints([[1, 2]] * 3), one), (x.t(), ints([[1]] * 50), one),
                 (x, ints([[1]] * 3), one, torch.zeros(2, device=DEV)), (x, ints([[1]] * 3), one, None, *k33),
                 (x, ints([[1]] * 3), one, None, k33[0][:, :4].contiguous()), (x[:, :0], ints([[1]] * 3), one)):
        with pytest.raises(kernels.KernelError):
            kernels.token_log_probs(*args)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 128), (F32, 64)])
def test_tree_attention_replayed_and_on_another_stream(dtype, d):
    c = drafted(13, [700, 130, 0], [9, 30, 1], 8, 2, d, 16, dtype)
    want = attend(c)
    out = torch.zeros_like(want)
    attend(c, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(c, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # other lengths in the same graph, within what the capture was told
    c["context"].copy_(ints([100, 33, 600]))
    table = torch.randperm(c["k"].shape[0], device=DEV)[:45].to(torch.int32)
    c["table"].copy_(table[:45].repeat(4)[:c["table"].numel()].view_as(c["table"]))
    c["k"].nan_to_num_(0.5), c["v"].nan_to_num_(0.5, 0.5, 0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, attend(c))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    again = torch.zeros_like(out)
    with torch.cuda.stream(side):
        attend(c, out=again)
    side.synchronize()
    assert torch.equal(out, again)


@pytest.mark.parametrize("name", ["clusters", "slices", "rows"])
def test_calls_on_two_streams_at_once(name):
    """Two kinds of work side by side give what each gives alone."""
    sizes = {"clusters": ([900, 300], [40, 9], 8, 2, 128, 16, BF), "slices": ([7000] * 12, [16] * 12, 32, 8, 64, 16, BF),
             "rows": ([500, 20], [7, 30], 8, 2, 64, 16, F32)}
    cases = [drafted(21, *sizes[name]), drafted(22, [1500, 7], [30, 60], 16, 2, 128, 16, BF)]
    alone = [attend(c) for c in cases]
    logits = torch.randn((40, 60000), device=DEV, generator=torch.Generator(DEV).manual_seed(3))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got, given = [[], []], []
    for _ in range(12):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(attend(cases[i]))
        with torch.cuda.stream(streams[2]):
            lp, ids, best = torch.empty((40, 1), device=DEV), torch.empty((40, 4), dtype=torch.int32, device=DEV), torch.empty((40, 4), device=DEV)
            kernels.token_log_probs(logits, torch.zeros((40, 1), dtype=torch.int32, device=DEV), lp, None, ids, best)
            given.append((lp, ids, best))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])
    values, order = logits.sort(dim=1, descending=True, stable=True)
    for lp, ids, best in given:
        assert torch.equal(ids.long(), order[:, :4]) and all(torch.equal(a, b) for a, b in zip((lp, ids, best), given[0]))


def test_tree_attention_a_chain_is_a_prompts_portion():
    """Drafted tokens without branches see what a portion of a prompt sees: the framework's own attention gives the same."""
    contexts, n = [211, 64, 5], 6
    c = drafted(14, contexts, [n] * 3, 8, 2, 128, 16, BF, chain=True)
    rows = c["q"].shape[0]
    out = torch.empty((rows, 8 * 128), dtype=BF, device=DEV)
    request = ints([r for r in range(3) for _ in range(n)])
    kernels.paged_attention_generic(c["q"], c["k"], c["v"], c["table"], request, c["positions"], 128 ** -0.5, 100, out)
    got = attend(c, 100)
    # the window slides over the drafted tokens too; here it is longer than the tree
    assert (got.float() - out.float()).abs().max() <= 2 * 2.0 ** -8 * out.float().abs().max() + 2.0 ** -8


# ---- what is moved ------------------------------------------------------------------------------------------------------
PAGES = [((3, 2, 9, 4, 16, 128), 2, BF), ((2, 9, 2, 16, 7), 1, F32), ((9, 1, 3, 5), 0, BF), ((2, 2, 9, 3, 16), 2, F32),
         ((2, 9, 3, 5, 3), 1, torch.uint8), ((4, 1, 9, 2, 16, 64), 2, torch.float8_e4m3fn), ((1, 9, 2, 64, 512), 1, F32)]


def raw(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    size = torch.empty((), dtype=dtype).element_size()
    return torch.randint(0, 256, shape[:-1] + (shape[-1] * size,), generator=g, dtype=torch.uint8).to(DEV).view(dtype)


@pytest.mark.parametrize("case", range(len(PAGES)))
def test_copied_pages(case):
    shape, axis, dtype = PAGES[case]
    pages = raw(shape, dtype)
    want = pages.clone().view(torch.uint8).flatten(0, axis - 1) if axis else pages.clone().view(torch.uint8)[None]
    source, target = [1, 1, 5, -1, 2, 3, 9, 7, 6], [0, 8, 4, 3, 9, -2, 3, 7, 6]
    for a, b in zip(source, target):
        if 0 <= a < 9 and 0 <= b < 9:
            want[:, b] = want[:, a]
    kernels.copy_pages(pages, axis, ints(source), ints(target))
    assert torch.equal(pages.view(torch.uint8).reshape(want.shape), want)
    kernels.copy_pages(pages, axis, ints([]), ints([]))
    assert torch.equal(pages.view(torch.uint8).reshape(want.shape), want)


@pytest.mark.parametrize("case", range(len(PAGES)))
@pytest.mark.parametrize("first", [0, 3, 20])
def test_kept_tokens(case, first):
    shape, axis, dtype = PAGES[case]
    places = shape[axis + 2]
    pages = raw(shape, dtype)
    rng = random.Random(case)
    table = torch.tensor([[4, 0, 7], [1, 8, -1], [3, 5, 2]], dtype=torch.int32)
    room = 3 * places - first
    sizes = [max(0, min(room, k)) for k in (room, 7, 0)]
    kept = [sorted(rng.sample(range(max(room, 1)), s)) if room > 0 else [] for s in sizes]
    kept[0] = kept[0][::2] if case % 2 else kept[0][1:]
    most = max(1, max(len(x) for x in kept))
    want = (pages.clone() if len(shape) > axis + 3 else pages.clone()[..., None]).view(torch.uint8)
    want = want.flatten(0, axis - 1) if axis else want[None]
    old = want.clone()
    for r, ks in enumerate(kept):
        for i, k in enumerate(ks):
            a, b = first + k, first + i
            pa, pb = (int(table[r, j // places]) if j // places < 3 else -1 for j in (a, b))
            if pa >= 0 and pb >= 0:
                want[:, pb, :, b % places] = old[:, pa, :, a % places]
    kernels.keep_tokens(pages, axis, table.to(DEV), ints([first] * 3), ints([x + [0] * (most - len(x)) for x in kept]),
                        ints([len(x) for x in kept]))
    assert torch.equal(pages.view(torch.uint8).reshape(want.shape), want)


@pytest.mark.parametrize("n,among", [(1000, 2000), (1999, 2000), (2000, 2000), (5, 3000), (1, 1)])
def test_many_kept_tokens(n, among):
    """Long runs, where a token's new place is another's old one many chunks ahead."""
    page, heads, d = 16, 2, 128
    count = -(-(among + 3) // page)
    pages = raw((2, count + 1, heads, page, d), BF)
    rng = random.Random(n)
    kept = sorted(rng.sample(range(among), n))
    order = list(range(count + 1))
    rng.shuffle(order)
    order = order[:count]
    flat = pages[:, order].transpose(2, 3).reshape(2, count * page, heads, d).clone()
    moved = flat.clone()
    moved[:, 3:3 + n] = flat[:, [3 + k for k in kept]]
    kernels.keep_tokens(pages, 1, ints([order]), ints([3]), ints([kept]), ints([n]))
    got = pages[:, order].transpose(2, 3).reshape(2, count * page, heads, d)
    assert torch.equal(got.view(torch.int16), moved.view(torch.int16))


# ---- log probabilities ---------------------------------------------------------------------------------------------------
def scored(logits, tokens, top, entropy=True):
    n = logits.shape[0]
    lp = torch.empty(tokens.shape, dtype=F32, device=DEV)
    h = torch.empty((n,), dtype=F32, device=DEV) if entropy else None
    ids = torch.full((n, top), -7, dtype=torch.int32, device=DEV) if top else None
    best = torch.empty((n, top), dtype=F32, device=DEV) if top else None
    kernels.token_log_probs(logits, tokens, lp, h, ids, best)
    return lp, h, ids, best


def same(got, want, vocab, big):
    """Within what 32-bit sums may be off.  S is a sum of positive numbers: each exponential is off by 2^-21 and its argument's
    2^-24 of itself (below 200, where the number counts for less than e^-200), the sum of n by (n / 512 + 40) roundings: its logarithm by
    that much; z by a rounding of the logits' magnitude (they differ by a rounding each), the result by one of its own."""
    off = 2.0 ** -20 + (vocab / 512 + 40) * 2.0 ** -24 + big * 2.0 ** -23
    got, want = got.cpu().double(), want.double()
    assert (torch.isnan(got) == torch.isnan(want)).all()
    assert (torch.isinf(got) == torch.isinf(want)).all()
    ok = torch.isfinite(want)
    assert ((got - want).abs() <= off + 2.0 ** -22 * want.abs())[ok].all(), (got - want).abs()[ok].max()


def compare(x, tokens, top):
    lp, h, ids, best = scored(x, tokens, top)
    wlp, wh, wids, wbest = plain.log_probs(x, tokens, top)
    vocab = x.shape[1]
    big = float(x.float().nan_to_num(0.0, 0.0, 0.0).abs().max())
    same(lp, wlp, vocab, big)
    # the entropy is log S - W / S, W a sum of as many numbers of one sign: off by as much, relative to itself, and S's share
    same(h, wh, vocab, big * 4)
    if top:
        assert torch.equal(ids.cpu().long(), wids)
        same(best, wbest, vocab, big)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,vocab,given,top", [
    (1, 151936, 1, 5), (3, 1000, 2, 32), (1, 1, 1, 1), (2, 7, 1, 32), (5, 33, 0, 2), (300, 517, 1, 20), (40, 8192, 3, 1), (2, 8193, 1, 0),
    (200, 20011, 1, 20), (7, 50001, 1, 31), (149, 32000, 1, 3), (1, 4097, 1, 8)])
def test_log_probs(dtype, rows, vocab, given, top):
    g = torch.Generator(device=DEV).manual_seed(vocab + rows)
    x = (3 * torch.randn((rows, vocab), generator=g, device=DEV)).to(dtype)
    t = torch.randint(0, vocab, (rows, given), generator=g, device=DEV).to(torch.int32)
    compare(x, t, top)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("skew", range(1, 9))
def test_log_probs_rows_that_lie_apart(dtype, skew):
    g = torch.Generator(device=DEV).manual_seed(skew)
    wide = torch.full((6, 5000 + 13), 1e4, device=DEV).to(dtype)
    x = wide[:, skew:skew + 5000]
    x.copy_(2 * torch.randn((6, 5000), generator=g, device=DEV))
    compare(x, torch.randint(0, 5000, (6, 2), generator=g, device=DEV).to(torch.int32), 9)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows", [2, 200])
def test_log_probs_hard_rows(dtype, rows):
    """Equal logits, ascending and descending ones, one above all, masked ones, infinities and no numbers."""
    vocab, inf, nan = 30000, float("inf"), float("nan")
    up = torch.arange(vocab, device=DEV, dtype=F32) / 1000
    kinds = [torch.zeros(vocab, device=DEV), torch.full((vocab,), -3.5, device=DEV), up, up.flip(0), torch.where(up == up[777], 90.0, 0.0),
             torch.where(up < 29.9, -inf, up), torch.where(up < 29.99, torch.finfo(dtype).min, up), torch.full((vocab,), -inf, device=DEV),
             torch.where(up == up[5], inf, up), torch.where(up == up[5], nan, up), torch.full((vocab,), nan, device=DEV),
             torch.where(up > 0.004, nan, up), torch.where(up > 0.004, -inf, -up), torch.where(up == 0, -0.0, 0.0), 1e4 + up, up * 1e30,
             torch.where(up.long() % 2 == 0, up, -up), torch.where(up < 12, up, 50 - up), up.flip(0).roll(9000)]
    x = torch.stack(kinds).to(dtype)
    x = x.repeat(-(-rows // len(kinds)), 1)[:max(rows, len(kinds))].contiguous()
    t = torch.randint(-3, vocab + 3, (x.shape[0], 4), device=DEV).to(torch.int32)
    t[:, 0] = 777
    lp, h, ids, best = scored(x, t, 20)
    wlp, wh, wids, wbest = plain.log_probs(x, t, 20)
    assert torch.equal(ids.cpu().long(), wids)
    for got, want in ((lp, wlp), (best, wbest), (h[:, None], wh[:, None])):
        for r in range(x.shape[0]):
            big = float(x[r].float().nan_to_num(0.0, 0.0, 0.0).abs().max())
            same(got[r], want[r], vocab, min(big, 1e5) * 4)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,vocab,given,top,skew", [
    (445, 1, 1, 1, 0), (445, 15, 40, 32, 1), (450, 16, 1, 16, 0), (446, 300, 1, 20, 3), (1001, 512, 2, 5, 7), (447, 513, 1, 32, 8), (500, 4089, 1, 8, 1),
    (500, 4090, 1, 8, 0), (445, 8185, 1, 32, 5), (445, 8186, 1, 3, 5), (3, 2048, 1, 8, 2), (1, 300, 1, 0, 3), (9, 2049, 3, 8, 1), (2, 40, 33, 8, 0)])
def test_log_probs_of_few_logits_a_row(dtype, rows, vocab, given, top, skew):
    g = torch.Generator(device=DEV).manual_seed(vocab + rows)
    wide = torch.full((rows, vocab + 9 + skew), 1e4, device=DEV).to(dtype)
    x = wide[:, skew:skew + vocab]
    x.copy_(3 * torch.randn((rows, vocab), generator=g, device=DEV))
    compare(x, torch.randint(0, vocab, (rows, given), generator=g, device=DEV).to(torch.int32), top)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab,top,rows", [(700, 20, 460), (700, 8, 19), (8000, 32, 460), (2000, 8, 460), (20, 32, 460)])
def test_log_probs_hard_rows_of_few_logits(dtype, vocab, top, rows):
    inf, nan = float("inf"), float("nan")
    at = torch.arange(vocab, device=DEV)
    up = at.to(F32) / 64
    kinds = [torch.zeros(vocab, device=DEV), torch.full((vocab,), -3.5, device=DEV), up, up.flip(0), torch.where(at == 7, 90.0, 0.0),
             torch.where(at < vocab - 5, -inf, up), torch.where(at < vocab - 5, torch.finfo(dtype).min, up), torch.full((vocab,), -inf, device=DEV),
             torch.where(at == 5, inf, up), torch.where(at == 5, nan, up), torch.full((vocab,), nan, device=DEV), torch.where(at > 4, nan, up),
             torch.where(at > 4, -inf, -up), torch.where(at == 0, -0.0, 0.0), 1e4 + up, up * 1e30, torch.where(at % 2 == 0, up, -up),
             torch.where(at % 16 == 3, 5.0, nan), up.flip(0).roll(vocab // 3)]
    x = torch.stack(kinds).to(dtype).repeat(-(-rows // len(kinds)), 1)[:rows].contiguous()
    t = torch.randint(-3, vocab + 3, (rows, 4), device=DEV).to(torch.int32)
    lp, h, ids, best = scored(x, t, top)
    wlp, wh, wids, wbest = plain.log_probs(x, t, top)
    assert torch.equal(ids.cpu().long(), wids)
    for got, want in ((lp, wlp), (best, wbest), (h[:, None], wh[:, None])):
        for r in range(rows):              # (rows that start elsewhere within 16 bytes are added up in another order)
            big = float(x[r].float().nan_to_num(0.0, 0.0, 0.0).abs().max())
            same(got[r], want[r], vocab, min(big, 1e5) * 4)


def test_log_probs_replayed():
    x = torch.randn((4, 40000), device=DEV)
    t = torch.randint(0, 40000, (4, 1), device=DEV).to(torch.int32)
    want = scored(x, t, 7)
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.token_log_probs(x, t, *outs)
    for _ in range(2):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- where keys and values go ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("dtype,d,value_is_key,norm", [(BF, 128, False, True), (BF, 128, True, True), (BF, 64, False, False), (BF, 80, True, False),
                                                       (F32, 128, False, True), (F32, 64, True, True)])
def test_keys_and_values_go_to_their_places(rows, dtype, d, value_is_key, norm):
    """With places a row's query, key and value are what they are without, and the key and value lie at the place."""
    g = torch.Generator().manual_seed(rows + d)
    nh, nkv, page = 4, 2, 16
    starts = [0, rows // 2, rows]
    request = [0] * (rows // 2) + [1] * (rows - rows // 2)
    positions = [i - starts[r] + 3 for i, r in enumerate(request)]
    places = []
    for r in range(2):                    # ascending, with gaps
        count = starts[r + 1] - starts[r]
        places += sorted(int(x) + 1 for x in torch.randperm(2 * count, generator=g)[:count])
    places[1] = -1                        # nowhere
    per = -(-(rows + 3) // page)
    table = torch.randperm(2 * per, generator=g).view(2, per).int().to(DEV)
    qkv = torch.randn((rows, (nh + nkv * (1 if value_is_key else 2)) * d), generator=g).to(dtype).to(DEV)
    weight = (1 + 0.1 * torch.randn((d,), generator=g)).to(dtype).to(DEV) if norm else None
    angle = torch.rand((rows + 3, d // 2), generator=g)
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)

    def run(at):
        k, v = torch.full((2 * per, nkv, page, d), 9.0, dtype=dtype, device=DEV), torch.full((2 * per, nkv, page, d), 9.0, dtype=dtype, device=DEV)
        q = torch.empty((rows, nh, d), dtype=dtype, device=DEV)
        kernels.qk_norm_rope_store(qkv, nh, nkv, d, True, weight, weight, 1e-6, cos, sin, d, ints(positions), ints(request), table, k, v, q,
                                   value_is_key=value_is_key, places=None if at is None else ints(at))
        return q, k, v

    q0, k0, v0 = run(None)
    assert all(torch.equal(a, b) for a, b in zip(run(positions), (q0, k0, v0)))
    q, k, v = run(places)
    assert torch.equal(q, q0)
    pages = table.cpu()
    written = torch.zeros((2 * per, page), dtype=torch.bool)
    for i, (r, p, a) in enumerate(zip(request, positions, places)):
        if a < 0:
            continue
        page0, page1 = int(pages[r, p // page]), int(pages[r, a // page])
        written[page1, a % page] = True
        assert torch.equal(k[page1, :, a % page], k0[page0, :, p % page]) and torch.equal(v[page1, :, a % page], v0[page0, :, p % page])
    # what lies behind a row's place in its page may be cleared; all else is as it was
    left = ~written.to(DEV)[:, None, :, None].expand_as(k)
    assert ((k == 9) | (k == 0))[left].all() and ((v == 9) | (v == 0))[left].all()
