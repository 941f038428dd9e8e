"""Calls in few bits right behind the kernels that write what they read, with the host far ahead of the device."""
from __future__ import annotations

import pytest
import torch

from test_few_bits_gpu import DT, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,kind", [(1, "bf16"), (5, "bf16"), (40, "bf16"), (300, "bf16"), (1, "f32"), (20, "f32"), (64, "f32"), (40, "mx4")])
@pytest.mark.parametrize("features,width", [(9000, 2048), (700, 5000)])
def test_a_product_right_behind_the_kernel_that_writes_its_weights(features, width, rows, kind):
    from inferrs_b200 import kernels as K
    x = rand((rows, width), 1).to(DT.get(kind, torch.bfloat16))
    given = K.quantize_mx4(x) if kind == "mx4" else x
    dense = [rand((features, width), 2 + i) for i in range(3)]
    want = []
    for d in dense:
        w = K.quantize_mx4(d)
        out = torch.empty((rows, features), device="cuda")
        torch.cuda.synchronize()
        K.linear_mx4(given, w, out)
        torch.cuda.synchronize()
        want.append(out)
    w = K.Mx4Matrix.empty(features, width, "cuda")
    got = [torch.empty_like(want[0]) for _ in range(60)]
    for start in range(0, 240, 60):
        torch.cuda._sleep(20_000_000)
        for i in range(60):
            K.quantize_mx4(dense[(start + i) % 3], out=w)
            K.linear_mx4(given, w, got[i])
        torch.cuda.synchronize()
        assert all(torch.equal(g, want[(start + i) % 3]) for i, g in enumerate(got))
    assert K.few_bits_faults() == {}
