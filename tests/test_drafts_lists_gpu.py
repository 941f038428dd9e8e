"""Attention of drafted tokens with lists that say too much: they are read as far as there are rows and places."""
from __future__ import annotations

import pytest
import torch

from inferrs_b200 import kernels
from test_drafts_gpu import BF, F32, attend, check, drafted, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(BF, 128), (BF, 64), (BF, 96), (F32, 64)])
def test_lists_that_say_too_much(dtype, d):
    """A first row before the first, a last one behind the last, a context of fewer than no tokens and one of more than the table has places."""
    c = drafted(16, [50, 7], [3, 4], 4, 2, d, 16, dtype)
    c["k"].nan_to_num_(0.5), c["v"].nan_to_num_(0.5, 0.5, 0.5)        # (places that held no key are places of the context now)
    got = attend(dict(c, q_start=ints([-5, 3, 2 ** 31 - 1]), context=ints([-3, 2 ** 31 - 1])))
    clipped = dict(c, q_start=ints([0, 3, 7]), context=ints([0, c["table"].shape[1] * 16]))
    check(clipped, got)
    assert torch.equal(got, attend(clipped))
    # the first request ends behind the last row, the second one before it begins
    c["most"] = 7
    assert torch.equal(attend(dict(c, q_start=ints([0, 9, 5]))), attend(dict(c, q_start=ints([0, 7, 7]))))
    assert kernels.attention_tree_error() == 0


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F32, 64)])
def test_windows_wider_than_any_context(dtype, d):
    c = drafted(16, [50, 300], [3, 4], 4, 2, d, 16, dtype)
    whole = attend(c)
    for span in (2 ** 31 - 1, 2 ** 31, 2 ** 31 + 5, 2 ** 40, 2 ** 32 + 7, -2 ** 31, -2 ** 32 - 9):
        assert torch.equal(attend(c, span), whole), span
