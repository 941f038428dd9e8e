"""What the calls for drafted tokens refuse, and the masks of trees (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from inferrs_b200 import kernels
from inferrs_b200.engine.batch import BatchError, tree_masks


def test_masks_of_trees():
    masks, depths = tree_masks([[-1, 0, 0, 1, -1], [], [-1] + list(range(33))])
    assert masks.dtype == np.int32 and masks.shape == (39, 2)
    assert masks[:5, 0].tolist() == [1, 3, 5, 11, 16] and (masks[:5, 1] == 0).all()
    assert depths[:5].tolist() == [0, 1, 1, 2, 0] and depths[5:].tolist() == list(range(34))
    assert masks[5 + 31].view(np.uint32).tolist() == [2 ** 32 - 1, 0] and masks[5 + 33].view(np.uint32).tolist() == [2 ** 32 - 1, 3]
    masks, _ = tree_masks([[-1]], words=3)
    assert masks.tolist() == [[1, 0, 0]]
    assert tree_masks([])[0].shape == (0, 1)
    for bad in ([0], [-1, 1], [-1, -2], [-1, 5]):
        with pytest.raises(BatchError):
            tree_masks([bad])
    with pytest.raises(BatchError):
        tree_masks([[-1] * 33], words=1)


def test_there_is_no_cpu_implementation():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)       # noqa: E731
    x = torch.zeros((2, 4, 16))
    pages = torch.zeros((3, 2, 4, 16))
    with pytest.raises(kernels.KernelError):
        kernels.paged_attention_tree(x, pages, pages, i(1, 2), i(2), i(1), i(2), i(2, 1), 1.0, None, torch.zeros((2, 64)), 2, 4)
    with pytest.raises(kernels.KernelError):
        kernels.copy_pages(pages, 0, i(1), i(1))
    with pytest.raises(kernels.KernelError):
        kernels.keep_tokens(pages, 0, i(1, 2), i(1), i(1, 2), i(1))
    with pytest.raises(kernels.KernelError):
        kernels.token_log_probs(torch.zeros((2, 9)), i(2, 1), torch.zeros((2, 1)))
