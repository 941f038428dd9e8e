"""Forks of every architecture and cache that the framework has, and which of them take drafted tokens."""
from __future__ import annotations

import importlib

import pytest
import torch

import test_few_bits_engine_gpu as few_bits
from helpers import PAGE_SIZE, random_tokens
from inferrs_b200.engine.batch import BatchError, DraftEntry, StepEntry

pytestmark = pytest.mark.gpu

FAMILIES = [(family, case) for family, cases in (("dasusun", "AC"), ("puposun", "AC"), ("ruzunex", "PQ"), ("sefalorn", "PQ"),
                                                 ("tikizen", "PQ"), ("vebonex", "PQ")) for case in cases]


def family_runner(family, case, dtype, **more):
    cases, tests = importlib.import_module(f"{family}_cases"), importlib.import_module(f"test_{family}_gpu")
    config = cases.CASES[case]
    if hasattr(cases, "for_dtype"):
        config = cases.for_dtype(config, dtype)
    return tests.make_runner(config, cases.make_weights(config, 7), dtype, n_pages=40, max_requests=3, **more)


def check_fork(make, n_prompt=61, n_more=6):
    """A request, its fork and a fork of the fork go different ways, step by step in turn: each has the bits of a request that ran the same
    steps without any fork.  The slots and pages have been another request's before."""
    runner, plain = make(), make()
    vocab = runner.spec.vocab_size
    prompt = random_tokens(n_prompt, vocab, seed=1)
    parts = [prompt[:37], prompt[37:]]
    ways = {r: random_tokens(n_more, vocab, seed=2 + i) for i, r in enumerate("abc")}

    def start(r, rid):
        r.admit(rid)
        for part in parts:
            r.step([StepEntry(rid, part, [len(part) - 1])])

    for rid in "xyz":                   # leftovers in every slot and in the pages
        runner.admit(rid)
        runner.step([StepEntry(rid, random_tokens(90, vocab, seed=ord(rid)), [])])
    for rid in "xyz":
        runner.release(rid)
    start(runner, "a")
    runner.fork("a", "b")
    runner.fork("b", "c")
    got = {r: [] for r in "abc"}
    for k in range(n_more):
        for r in "abc":
            got[r].append(runner.step([StepEntry(r, [ways[r][k]], [0])]).clone())
    runner.manager.check_invariants()
    for r in "abc":
        start(plain, r)
        for k in range(n_more):
            want = plain.step([StepEntry(r, [ways[r][k]], [0])])
            assert torch.isfinite(want).all() and torch.equal(got[r][k], want), (r, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("family,case", FAMILIES)
def test_forks_of_every_architecture(family, case, dtype):
    check_fork(lambda: family_runner(family, case, dtype))


@pytest.mark.parametrize("family", ["vebonex", "puposun"])
def test_forks_beside_replayed_steps(family):
    case = "P" if family == "vebonex" else "A"
    check_fork(lambda: family_runner(family, case, torch.bfloat16, use_graphs=True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("weight_bits", [None, 4])
def test_forks_over_the_cache_in_8_bits(model_dirs, dtype, weight_bits):
    check_fork(lambda: few_bits.make_runner(model_dirs["D"], dtype, "D", weight_bits, 8))


@pytest.mark.parametrize("family,case", FAMILIES)
def test_models_that_take_no_drafts_say_so(family, case):
    """Layers with a state of fixed size, latents, kept first keys, shaped scores, values of their own: a tree is refused before anything is taken."""
    runner = family_runner(family, case, torch.float32)
    runner.admit(0)
    runner.step([StepEntry(0, [1, 2, 3], [])])
    free = [p.n_free for p in runner.manager.pools]
    assert not runner.takes_drafts()
    with pytest.raises(BatchError):
        runner.step_drafts([DraftEntry(0, [4], [-1])])
    assert [p.n_free for p in runner.manager.pools] == free and runner.n_tokens(0) == 3


def test_the_cache_in_8_bits_takes_no_drafts(model_dirs):
    runner = few_bits.make_runner(model_dirs["D"], torch.bfloat16, "D", None, 8)
    runner.admit(0)
    assert not runner.takes_drafts()
    with pytest.raises(BatchError):
        runner.step_drafts([DraftEntry(0, [4], [-1])])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafts_with_weights_in_4_bits(model_dirs, dtype):
    """Only the cache's type decides: a chain of drafted tokens through 4-bit weights gives what the tokens one after another give."""
    runner = few_bits.make_runner(model_dirs["D"], dtype, "D", 4, None)
    assert runner.takes_drafts()
    vocab = runner.spec.vocab_size
    prompt, chain = random_tokens(2 * PAGE_SIZE["D"] + 3, vocab, seed=5), random_tokens(5, vocab, seed=6)
    for rid in (0, 1):
        runner.admit(rid)
        runner.step([StepEntry(rid, prompt, [])])
    got = runner.step_drafts([DraftEntry(0, chain, [-1, 0, 1, 2, 3])])
    want = torch.cat([runner.step([StepEntry(1, [t], [0])]).clone() for t in chain])
    assert float((got - want).abs().max() / want.abs().max()) < few_bits_bound(dtype)


def few_bits_bound(dtype):
    return {torch.float32: 1e-4, torch.bfloat16: 3e-2}[dtype]      # the same sums in another order (test_engine_gpu.py)
