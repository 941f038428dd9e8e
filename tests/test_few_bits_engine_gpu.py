"""A model in few bits through the engine: weights in 4 bits, the cache in 8, both, against the plain implementation with the same
numbers (weights replaced by what they stand for in 4 bits, keys and values by what they stand for in 8)."""
from __future__ import annotations

import pytest
import torch

import plain_few_bits
import plain_qwen3
from helpers import CONFIG_A, CONFIG_C, CONFIG_D, PAGE_SIZE, cut, random_tokens, rel_err
from inferrs_b200 import Engine, SamplingParams
from inferrs_b200.engine.batch import StepEntry
from inferrs_b200.engine.loading import load_model_dir
from inferrs_b200.engine.runner import ModelRunner
from inferrs_b200.runtime import Runtime

pytestmark = pytest.mark.gpu
CONFIGS = {"A": CONFIG_A, "C": CONFIG_C, "D": CONFIG_D}
BITS = [(4, None), (None, 8), (4, 8)]


def tolerance(dtype, cache_bits):
    """Without a cache in few bits the engine's own (the arithmetic is the same but for the weights' values).  With it, a key or
    value whose last bits differ may fall to the next code, 2^-4 of it away: rare in float32, common where rows are rounded
    to bfloat16 in between."""
    return (5e-3 if cache_bits else 1e-4) if dtype == torch.float32 else (6e-2 if cache_bits else 3e-2)


def plain_logits(model_dir, tokens, dtype, weight_bits, cache_bits, monkeypatch):
    cfg, w = plain_qwen3.read_model(model_dir)
    if weight_bits:
        store = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
        w = {k: plain_few_bits.values4(v.to(store))[0].float() if k.endswith("_proj.weight") else v for k, v in w.items()}
    if cache_bits:
        attention = plain_qwen3.causal_attention

        def in_eight_bits(q, k, v, scale, window=None):
            k, v = (codes * s.unsqueeze(-1) for codes, s in (plain_few_bits.to8(t.double()) for t in (k, v)))
            return attention(q, k.float(), v.float(), scale, window)

        monkeypatch.setattr(plain_qwen3, "causal_attention", in_eight_bits)
    out = plain_qwen3.forward(cfg, w, tokens, store=None if dtype == torch.float32 else dtype)
    monkeypatch.undo()
    return out


def make_runner(model_dir, dtype, name, weight_bits, cache_bits, n_pages=64, **more):
    rt = Runtime.cuda(dtype, weight_bits, cache_bits)
    spec, weights, _ = load_model_dir(model_dir, rt)
    return ModelRunner(spec, weights, rt, page_size=PAGE_SIZE[name], n_pages=n_pages, max_requests=4, **more)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["A", "C", "D"])
def test_logits_in_portions_and_one_by_one(model_dirs, name, dtype, bits, monkeypatch):
    toks = random_tokens(131, CONFIGS[name]["vocab_size"], seed=12)
    want = plain_logits(model_dirs[name], toks, dtype, *bits, monkeypatch)
    runner = make_runner(model_dirs[name], dtype, name, *bits)
    runner.admit("r")
    rows, at = [], 0
    for n in cut(99, [40, 2, 13, 3, 1]) + [1] * 32:
        rows.append(runner.step([StepEntry("r", toks[at:at + n], list(range(n)))]))
        at += n
    err = rel_err(torch.cat(rows).cpu(), want)
    assert err < tolerance(dtype, bits[1]), err
    from inferrs_b200 import kernels
    assert kernels.few_bits_faults() == {}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_requests_beside_one_another_and_pages_used_again(model_dirs, dtype, monkeypatch):
    lens = [70, 23, 97, 31, 18, 64]
    prompts = [random_tokens(n, CONFIG_D["vocab_size"], seed=20 + i) for i, n in enumerate(lens)]
    runner = make_runner(model_dirs["D"], dtype, "D", 4, 8, n_pages=18)
    want = [plain_logits(model_dirs["D"], p, dtype, 4, 8, monkeypatch) for p in prompts]
    for pair in ((0, 1), (2, 3), (4, 5)):
        for i in pair:
            runner.admit(i)
        at = {i: 0 for i in pair}
        got = {i: [] for i in pair}
        while any(at[i] < lens[i] for i in pair):
            entries = []
            for i in pair:
                n = min((1, 9, 17)[(at[i] + i) % 3], lens[i] - at[i])
                if n:
                    entries.append(StepEntry(i, prompts[i][at[i]:at[i] + n], list(range(n))))
            rows = runner.step(entries)
            done = 0
            for e in entries:
                got[e.rid].append(rows[done:done + len(e.tokens)])
                done += len(e.tokens)
                at[e.rid] += len(e.tokens)
        for i in pair:
            assert rel_err(torch.cat(got[i]).cpu(), want[i]) < tolerance(dtype, 8)
            runner.release(i)


@pytest.mark.parametrize("bits", BITS)
def test_replayed_steps_give_what_plain_launches_give(model_dirs, bits):
    toks = random_tokens(120, CONFIG_D["vocab_size"], seed=3)
    out = []
    for graphs in (False, True):
        runner = make_runner(model_dirs["D"], torch.bfloat16, "D", *bits, use_graphs=graphs)
        runner.admit("r")
        rows, at = [], 0
        for n in (64, 1, 1, 32, 1, 1, 16, 4):
            rows.append(runner.step([StepEntry("r", toks[at:at + n], [n - 1])]).clone())
            at += n
        out.append(torch.cat(rows))
    assert rel_err(out[1].cpu(), out[0].cpu()) < tolerance(torch.bfloat16, bits[1])


def test_generation_through_the_engine_and_its_memory(model_dirs):
    """Tokens in float32 are those of a model whose weights hold the 4-bit values; the cache counts its own bytes."""
    prompts = [random_tokens(n, CONFIG_D["vocab_size"], seed=n) for n in (70, 5, 33)]
    eng = Engine(model_dirs["D"], dtype="f32", block_size=16, num_blocks=32, max_batch_size=4, weight_bits=4)
    got = eng.generate(prompts, SamplingParams.greedy(max_tokens=6))
    cfg, w = plain_qwen3.read_model(model_dirs["D"])
    w = {k: plain_few_bits.values4(v)[0].float() if k.endswith("_proj.weight") else v for k, v in w.items()}
    for p, tokens in zip(prompts, got):
        toks = list(p)
        for t in tokens:
            assert int(plain_qwen3.forward(cfg, w, toks)[-1].argmax()) == t
            toks.append(t)
    both = Engine(model_dirs["D"], dtype="bf16", block_size=16, num_blocks=32, max_batch_size=4, weight_bits=4, cache_bits=8)
    assert all(len(t) == 6 for t in both.generate(prompts, SamplingParams.greedy(max_tokens=6)))
    assert both.runner.storage.bytes_per_token() == 2 * 2 * 2 * (128 + 4)       # layers, keys and values, heads
    assert both.stats()["kernel_errors"] == []


def test_what_has_no_form_in_few_bits_refuses(model_dirs):
    from inferrs_b200.engine.model import ModelError
    from inferrs_b200.engine.loading import random_model
    from tikizen_cases import CASE_P
    with pytest.raises(ValueError):
        Runtime.cuda("bf16", weight_bits=3)
    with pytest.raises(ValueError):
        Runtime.cuda("bf16", cache_bits=4)
    for bits in ((4, None), (None, 8)):
        rt = Runtime.cuda("bf16", *bits)
        spec, weights, _ = random_model(CASE_P, 0, rt)
        with pytest.raises((ModelError, ValueError)):
            ModelRunner(spec, weights, rt, page_size=16, n_pages=8, max_requests=2)


def test_command_line_in_few_bits(model_dirs, capsys):
    from inferrs_b200.cli import main
    assert main(["run", model_dirs["D"], "--prompt-ids", "1,2,3", "--max-tokens", "4", "--temperature", "0", "--max-blocks", "8",
                 "--weight-bits", "4", "--cache-bits", "8", "--ignore-eos"]) == 0
    assert len(capsys.readouterr().out.split()) == 4
