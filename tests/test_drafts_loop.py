"""Scores of prompts beside live requests, on the CPU: the engine's loop with a stand-in for the model (test_engine_loop.py)."""
from __future__ import annotations

import pytest
import torch

from inferrs_b200.engine.engine import KernelFault
from inferrs_b200.sampling.params import SamplingParams
from test_engine_loop import VOCAB, FakeHealth, make_engine, plain_generate


def engine(overlap, fail_at=None):
    eng, manager = make_engine(overlap, n_pages=64, page_size=4, slots=4, max_batch=3, budget=16, chunk=None, eos=())
    eng.runner.admit, eng.runner.release = manager.admit, manager.release
    eng._scores = lambda logits, tokens, top: torch.zeros((logits.shape[0], 2 + 2 * top))
    if fail_at is not None:
        eng.health = FakeHealth(fail_at, every=10 ** 9)
    return eng, manager


def finish(eng, done):
    for _ in range(500):
        if not eng.has_work():
            break
        for r in eng.step():
            assert r.rid not in done
            done[r.rid] = r
    for r in eng.flush():
        done[r.rid] = r


@pytest.mark.parametrize("overlap", [False, True])
@pytest.mark.parametrize("pending", [False, True])
def test_scores_look_at_what_the_kernels_report(overlap, pending):
    """A word that was set while prompts were scored is found by the call itself, also where a look was already on its way (which says
    nothing of what came behind it); the live requests end with it and the next step says so."""
    prompts = [[1, 2, 3], [4, 5, 6, 7, 8]]
    eng, manager = engine(overlap, fail_at=0)
    out = eng.score(prompts)
    assert [len(x) for x in out] == [2, 4] and eng.health.asked == 1 and not eng.health.pending

    eng, manager = engine(overlap, fail_at=2 if pending else 1)
    live = SamplingParams(temperature=0.0, max_tokens=30)
    for i in range(2):
        eng.add_request([1 + i, 2, 3], live, rid=i)
    for _ in range(3):
        assert eng.step() == []
    if pending:
        eng.health.queue()
    with pytest.raises(KernelFault):
        eng.score(prompts)
    assert eng.health.n_reset == 1 and len(eng.kernel_errors) == 1 and not eng.health.pending
    assert eng.has_work() and manager.n_live == 0
    done = {}
    eng.add_request([9, 9], SamplingParams(temperature=0.0, max_tokens=4), rid=2)
    finish(eng, done)
    assert sorted(done) == [0, 1, 2] and done[0].finish_reason == done[1].finish_reason == "error"
    assert (done[2].output, done[2].finish_reason) == plain_generate([9, 9], SamplingParams(temperature=0.0, max_tokens=4), ())
    assert manager.pools[0].n_free == 64


@pytest.mark.parametrize("overlap", [False, True])
def test_scores_beside_live_requests_change_nothing(overlap):
    eng, manager = engine(overlap, fail_at=0)
    params = [SamplingParams(temperature=0.0, max_tokens=n) for n in (3, 12, 7)]
    prompts = [[(5 * i + j) % VOCAB for j in range(4 + 9 * i)] for i in range(3)]
    for i, (p, sp) in enumerate(zip(prompts, params)):
        eng.add_request(p, sp, rid=i)
    done = {}
    for _ in range(4):
        for r in eng.step():
            done[r.rid] = r
        assert [len(x) for x in eng.score([[7], [1, 2], list(range(20))])] == [0, 1, 19]
    finish(eng, done)
    for i in range(3):
        assert (done[i].output, done[i].finish_reason) == plain_generate(prompts[i], params[i], ())
    manager.check_invariants()


def test_generation_looks_behind_its_last_step():
    """A look that was on its way before the last step says nothing of that step: the one at the end is asked for behind it."""
    eng, _ = engine(False, fail_at=2)
    eng.health.every = 1
    asked = []
    queue = eng.health.queue

    def queued():
        asked.append(eng.n_steps)
        queue()

    eng.health.queue = queued
    eng.health.poll = lambda wait=False, poll=eng.health.poll: poll(wait) if wait else None      # (the first answer never comes by itself)
    with pytest.raises(KernelFault):
        eng.generate([[1, 2, 3]], SamplingParams(temperature=0.0, max_tokens=6))
    assert asked == [1, eng.n_steps]


def test_how_many_of_the_likeliest_tokens_can_be_asked_for():
    """A number that is none is refused where it is given, not in the middle of a step that other requests share."""
    for good in (0, 1, 32, torch.tensor(3)):
        assert SamplingParams(logprobs=good).logprobs == int(good) and type(SamplingParams(logprobs=good).logprobs) is int
    assert SamplingParams().logprobs is None
    eng, manager = engine(False)
    for bad in (-1, 33, 2.5, 2.0, "3", [1]):
        with pytest.raises(ValueError):
            SamplingParams(logprobs=bad)
        with pytest.raises(ValueError):
            eng.score([[1, 2]], top=bad)


def test_a_prompt_to_score_is_checked_before_anything_runs():
    """Also its last token, which no step runs where the tokens ahead of it fill whole portions."""
    eng, manager = engine(False)
    portion = eng.scheduler.max_tokens_per_step
    for prompt in ([1] * portion + [VOCAB], [1, VOCAB, 2], [-1, 2]):
        with pytest.raises(ValueError):
            eng.score([[1, 2, 3], prompt])
    assert eng.runner.hash == {} and manager.n_live == 0
    assert eng.score([[], [1]]) == [[], []]
