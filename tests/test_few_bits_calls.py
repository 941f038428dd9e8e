"""Which calls an attention layer over a cache in 8 bits makes in a step, and what the options' arguments keep of older calls (no GPU)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from inferrs_b200 import kernels
from inferrs_b200.parts.attention import Attention
from inferrs_b200.runtime import Runtime


def calls_of_a_step(monkeypatch, head_dim, page_size, q_lens, dtype=torch.bfloat16):
    """The tiles (None: rows one by one) of each attention call of a step of these portions, 8 heads on 2."""
    calls = []
    monkeypatch.setattr(kernels, "qk_norm_rope_store_kv8", lambda *a, **k: None)
    monkeypatch.setattr(kernels, "paged_attention_kv8", lambda *a, tiles=None: calls.append(tiles))
    layer = Attention.__new__(Attention)
    layer.spec = SimpleNamespace(n_heads=8, n_kv_heads=2, head_dim=head_dim, scale=1.0)
    layer.rt, layer.span = SimpleNamespace(dtype=dtype), None
    for name in ("q_weight", "k_weight", "eps", "cos", "sin", "rot_dim", "interleaved"):
        setattr(layer, name, None)
    pages = SimpleNamespace(k=torch.empty((4, 2, page_size, head_dim), dtype=torch.uint8))
    n, singles = sum(q_lens), [x for x in q_lens if x == 1]
    ctx = SimpleNamespace(storage=SimpleNamespace(pages8=lambda _: (pages, 0)), block_tables=[None], positions=None, row_request=None,
                          q_start=None, max_kv_len=n, n_rows=n, extra={}, decode_only=max(q_lens) == 1,
                          single_rows=lambda: ("rows", "reqs", len(singles)),
                          attention_tiles=lambda tokens, portions_only: ("req", "row0", -(-n // tokens)))
    layer._attend_kv8(ctx, 0, torch.empty((n, 12 * head_dim)), None)
    return calls


@pytest.mark.parametrize("head_dim,page_size", [(128, 8), (128, 24), (64, 4), (80, 16), (256, 40)])
def test_what_the_tensor_cores_kernels_do_not_take_is_one_call(monkeypatch, head_dim, page_size):
    """Pages of other than 16 places and other heads go row by row in every call: two calls would do every row twice."""
    assert calls_of_a_step(monkeypatch, head_dim, page_size, [1, 900, 1, 700]) == [None]


def test_portions_go_in_tiles_and_single_tokens_beside_large_ones_by_themselves(monkeypatch):
    assert calls_of_a_step(monkeypatch, 128, 16, [1, 900, 1, 700]) == [("reqs", "rows", 2, None, 1), ("req", "row0", 26, None, 64)]
    assert calls_of_a_step(monkeypatch, 128, 32, [1, 30]) == [("req", "row0", 4, None, 8)]
    assert calls_of_a_step(monkeypatch, 128, 16, [1, 1]) == [None]
    assert calls_of_a_step(monkeypatch, 128, 16, [1, 900], torch.float32) == [None]


def test_a_runtime_takes_its_arguments_in_the_order_that_it_had():
    """The tables that parts share came third before there were options in few bits."""
    tables = {"a": 1}
    rt = Runtime(torch.device("cpu"), torch.float32, tables)
    assert rt.shared is tables and rt.weight_bits is None and rt.cache_bits is None
    rt = Runtime(torch.device("cpu"), torch.float32, weight_bits=4, cache_bits=8)
    assert rt.shared == {} and (rt.weight_bits, rt.cache_bits) == (4, 8)
    for bad in (dict(weight_bits=8), dict(cache_bits=4)):
        with pytest.raises(ValueError):
            Runtime(torch.device("cpu"), torch.float32, **bad)


def test_a_matrix_in_four_bits_is_on_a_gpu():
    for device in ("cpu", torch.device("cpu"), "meta"):
        with pytest.raises(kernels.KernelError):
            kernels.Mx4Matrix.empty(4, 64, device)
