"""Drafted tokens and forks through the runner on the CPU, with plain statements in the kernels' place."""
from __future__ import annotations

import random

import pytest
import torch

import drafts_refs
import plain_qwen3
from helpers import CONFIG_A, CONFIG_B, PAGE_SIZE, random_tokens, rel_err
from inferrs_b200.cache.manager import CacheError, CacheManager, GroupLayout, OutOfPages
from inferrs_b200.engine.batch import BatchError, DraftEntry, StepEntry
from inferrs_b200.engine.loading import load_model_dir
from inferrs_b200.engine.runner import ModelRunner
from inferrs_b200.runtime import Runtime

CONFIGS = {"A": CONFIG_A, "B": CONFIG_B}


def make_runner(model_dir, page_size, n_pages=32, max_requests=3):
    rt = Runtime(torch.device("cpu"), torch.float32)
    spec, weights, _ = load_model_dir(model_dir, rt)
    return ModelRunner(spec, weights, rt, page_size=page_size, n_pages=n_pages, max_requests=max_requests)


def last_logits(model_dir, tokens):
    cfg, w = plain_qwen3.read_model(model_dir)
    return plain_qwen3.forward(cfg, w, tokens)[-1]


def pages_held(runner, rid):
    return [len(runner.manager.block_table(rid, g)) for g in range(len(runner.manager.groups))]


# ---- pages that were taken for tokens that never came -------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(6))
def test_the_book_takes_back_what_is_not_needed(seed):
    rng = random.Random(seed)
    page = rng.choice([1, 4, 16])
    m = CacheManager([GroupLayout("full"), GroupLayout("window", window=rng.choice([1, 7, 40]))], page, [60, 60], 4)
    held, taken = {}, {}
    for _ in range(200):
        rid = rng.randrange(4)
        if not m.has(rid):
            m.admit(rid)
            held[rid] = taken[rid] = 0
        what = rng.random()
        if what < 0.5:
            n = rng.randrange(1, 30)
            try:
                m.reserve({rid: n})
            except OutOfPages:
                continue
            taken[rid] = max(taken[rid], held[rid] + n)
        elif what < 0.8:
            n = rng.randrange(0, 20)
            free = [p.n_free for p in m.pools]
            m.trim(rid, n)
            after = max(0, -(-taken[rid] // page) - -(-(held[rid] + n) // page))
            assert m.pools[0].n_free == free[0] + after
            assert m.pools[1].n_free >= free[1]
            taken[rid] = min(taken[rid], -(-(held[rid] + n) // page) * page)
            with pytest.raises(CacheError):
                m.commit(rid, n + 1)
        elif what < 0.95:
            try:
                m.commit(rid, 1)
                held[rid] += 1
            except CacheError:
                pass
        else:
            m.release(rid)
        m.check_invariants()
        for r in range(4):
            if m.has(r):
                assert m.n_tokens(r) == held[r] and len(m.block_table(r, 0)) == -(-max(taken[r], held[r]) // page)
    with pytest.raises(CacheError):
        m.trim("nobody", 1)
    for r in range(4):
        if m.has(r):
            with pytest.raises(CacheError):
                m.trim(r, -1)
            m.release(r)
    assert [p.n_free for p in m.pools] == [60, 60]


@pytest.mark.parametrize("name", ["A", "B"])
def test_pages_of_drafts_that_are_not_kept_come_back(model_dirs, monkeypatch, name):
    """A request holds the pages of what it holds: behind a tree of which some or none was kept, behind a step that wrote over a tree, and
    behind a call that was refused (where an earlier tree may still be kept)."""
    drafts_refs.install(monkeypatch)
    page, vocab = PAGE_SIZE[name], CONFIGS[name]["vocab_size"]
    runner = make_runner(model_dirs[name], page)
    prompt = random_tokens(page + 1, vocab, seed=1)
    runner.admit(0)
    runner.step([StepEntry(0, prompt, [])])
    groups = len(runner.manager.groups)
    tree = [-1] + [0] * (2 * page)
    drafts = random_tokens(len(tree), vocab, seed=2)
    assert pages_held(runner, 0) == [2] * groups
    logits = runner.step_drafts([DraftEntry(0, drafts, tree)])
    for i in (0, 1, len(tree) - 1):
        tokens = prompt + [drafts[0]] + ([drafts[i]] if i else [])
        assert rel_err(logits[i], last_logits(model_dirs[name], tokens)) < 1e-4
    wide = -(-(page + 1 + len(tree)) // page)
    assert pages_held(runner, 0) == [wide] * groups
    with pytest.raises(BatchError):
        runner.step_drafts([DraftEntry(0, [vocab], [-1])])
    with pytest.raises(BatchError):
        runner.step_drafts([DraftEntry(0, [1] * (5 * page), [-1] + [3] * (5 * page - 1))])
    assert pages_held(runner, 0) == [wide] * groups
    runner.keep_drafts({0: [0, len(tree) - 1]})
    assert runner.n_tokens(0) == page + 3 and pages_held(runner, 0) == [-(-(page + 3) // page)] * groups
    held = prompt + [drafts[0], drafts[-1]]
    runner.step_drafts([DraftEntry(0, drafts, tree)])
    got = runner.step([StepEntry(0, [5], [0])])                # nobody kept them
    assert rel_err(got[0], last_logits(model_dirs[name], held + [5])) < 1e-4
    assert pages_held(runner, 0) == [-(-(page + 4) // page)] * groups
    runner.step_drafts([DraftEntry(0, drafts, tree)])
    runner.step_drafts([DraftEntry(0, [7], [-1])])             # a smaller tree in the place of a larger one
    assert pages_held(runner, 0) == [-(-(page + 5) // page)] * groups
    runner.keep_drafts({0: []})
    assert pages_held(runner, 0) == [-(-(page + 4) // page)] * groups
    got = runner.step([StepEntry(0, [6], [0])])
    assert rel_err(got[0], last_logits(model_dirs[name], held + [5, 6])) < 1e-4
    runner.manager.check_invariants()


def test_a_step_without_room_leaves_drafts_that_can_be_kept(model_dirs, monkeypatch):
    drafts_refs.install(monkeypatch)
    page = PAGE_SIZE["A"]
    runner = make_runner(model_dirs["A"], page, n_pages=4)
    for i in range(2):
        runner.admit(i)
    runner.step([StepEntry(0, [1] * page, []), StepEntry(1, [2] * page, [])])
    runner.step_drafts([DraftEntry(0, [5] * page, [-1] + [0] * (page - 1))])
    with pytest.raises(OutOfPages):
        runner.step([StepEntry(0, [3], [0]), StepEntry(1, [4] * (page + 1), [0])])
    with pytest.raises(OutOfPages):
        runner.step_drafts([DraftEntry(0, [3], [-1]), DraftEntry(1, [4] * (page + 1), [-1] * (page + 1))])
    runner.keep_drafts({0: [0, page - 1]})
    assert runner.n_tokens(0) == page + 2
    runner.manager.check_invariants()
