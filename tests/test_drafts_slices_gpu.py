"""Attention of drafted tokens whose keys are cut into slices: spans that leave some requests fewer slices than others, against the definition
in 64 bits."""
from __future__ import annotations

import pytest

import plain_drafts as plain
from inferrs_b200 import kernels
from test_drafts_gpu import BF, attend, check, drafted

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert kernels.attention_tree_error() == 0


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("most", [40, 9])       # two sets of rows a CTA, and one
@pytest.mark.parametrize("span,ahead", [(-3200, 0), (-1600, 0), (7000, 7000), (7000, 100000), (7000, 3000)])
def test_spans_that_leave_few_slices(d, most, span, ahead):
    """Chunks that begin shortly before some contexts end, and windows that have left most of a context behind: of a request's slices
    one may be left, or some, while others have them all."""
    contexts = [3200, 3201, 3330, 6400, 3199, 9, 0, 6399, 5000, 3300]
    trees = [most, 1, 33 if most > 33 else 3, most, 2, most, 1, most - 1, 5, most]
    c = drafted(41, contexts, trees, 32, 8, d, 16, BF, chain=ahead == 3000, spare=1)
    c["positions"] = c["positions"] + ahead
    c["longest"] = 16448            # (as many slices as such a request would have)
    check(c, attend(c, span), span)


def workspace(requests, tree, longest, heads, kv, d, span=0):
    """The bytes that the call asks for (nothing is read)."""
    return kernels._drafts().ib_paged_attention_tree_workspace(kernels._TREE_CALL(
        *[0] * 11, 0, heads * d, requests * tree, requests, heads, kv, d, -(-longest // 16), 16, 1 << 20, -(-tree // 32), span, tree, longest, d ** -0.5))


def test_the_workspace_is_bounded_and_goes_by_the_rows_in_use():
    for requests in (10, 16, 64, 256, 1024):
        for tree in (1, 4, 8, 40, 64, 128):
            for longest in (7000, 16384, 131072, 1 << 20):
                for heads, kv, d in ((32, 8, 128), (64, 8, 128), (32, 8, 64), (16, 8, 128)):
                    assert 0 <= workspace(requests, tree, longest, heads, kv, d) <= 256 << 20, (requests, tree, longest, heads, d)
    # trees of four tokens, four heads a group: 16 rows, 32 lines in each of two streams, and not 256 lines
    one = workspace(10, 4, 16384, 32, 8, 128)
    slices = -(-(16384 // 128) // 24)
    assert one == 10 * 8 * slices * (2 * 32 * (128 + 2) + 4) * 4
    # the largest of the benchmarked ones has what it had
    assert workspace(16, 64, 16384 + 64, 32, 8, 128) == 16 * 8 * 6 * (256 * (128 + 2) + 4) * 4


@pytest.mark.parametrize("d,requests,span", [(128, 40, None), (128, 300, None), (64, 80, None), (64, 80, 9000), (64, 600, None)])
def test_many_requests_with_one_of_them_long(d, requests, span):
    """The bound on the workspace leaves the long request fewer and longer slices than there could be, or none at all."""
    long = {40: 20000, 80: 20000}.get(requests, 6300)
    contexts, trees = [5 + i % 9 for i in range(requests)], [1 + i % 2 for i in range(requests)]
    contexts[1], trees[1], trees[2] = long, 3, 40
    contexts[3], trees[3] = 3500, 2
    c = drafted(51, contexts, trees, 32, 8, d, 16, BF)
    c["longest"] = 131072
    check(c, attend(c, span), span)


def test_trees_that_are_larger_than_the_call_says():
    """Rows beyond ``max_tree`` may be left out, and are if there is no room for their sums; the others are right."""
    contexts, trees = [6400, 3200, 9, 0, 3000, 40, 3, 7, 9, 10], [40, 9, 1, 40, 9, 2, 9, 9, 30, 9]
    c = drafted(61, contexts, trees, 32, 8, 128, 16, BF)
    want, off = plain.tree_attention(c["q"], c["k"], c["v"], c["table"], c["q_start"], c["context"], c["positions"], c["seen"], 128 ** -0.5, 0)
    c["most"] = 9
    got = attend(c).cpu().view(want.shape)
    right = ((got.double() - want).abs() <= off + plain.HALF[BF] * (want.abs() + off)).flatten(1).all(1)
    start = c["q_start"].tolist()
    for r in range(len(trees)):
        rows = slice(start[r], start[r + 1])
        assert right[rows][:9].all() and (right[rows] | (got[rows] == 7.0).flatten(1).all(1)).all()


@pytest.mark.parametrize("requests", [63, 64, 65, 130])
def test_requests_in_order_of_their_length_and_as_they_come(requests):
    """The CTAs of few requests take the longest ones first, those of more take them as they come; equal lengths among both."""
    contexts = [(i * 37) % 11 * 40 for i in range(requests)]
    trees = [1 + i % 5 for i in range(requests)]
    c = drafted(71, contexts, trees, 8, 4, 128, 16, BF)
    check(c, attend(c))
