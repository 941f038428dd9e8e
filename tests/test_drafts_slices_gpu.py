"""Attention of drafted tokens whose keys are cut into slices: spans that leave some requests fewer slices than others, against the definition
in 64 bits."""
from __future__ import annotations

import pytest
import torch

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
