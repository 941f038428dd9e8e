"""Drafted tokens and forks through the runner on the CPU, with plain statements in the kernels' place."""
from __future__ import annotations

import dataclasses
import random

import pytest
import torch

import drafts_refs
import plain_qwen3
from helpers import CONFIG_A, CONFIG_B, PAGE_SIZE, random_tokens, rel_err
from inferrs_b200.cache.manager import CacheError, CacheManager, GroupLayout, OutOfPages
from inferrs_b200.engine.batch import BatchError, DraftEntry, StepEntry
from inferrs_b200.engine.loading import load_model_dir, spec_from_config
from inferrs_b200.engine.model import declared_tensors
from inferrs_b200.engine.runner import ModelRunner
from inferrs_b200.parts.spec import ScheduleEntry
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


# ---- forks --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(8))
def test_the_book_of_a_fork(seed):
    """A fork has as many tokens, its own pages where the other one has pages, and none where a window has passed; it needs no room beyond that."""
    rng = random.Random(100 + seed)
    page = rng.choice([1, 4, 16])
    window, keep = rng.choice([1, 7, 40]), rng.choice([0, 5])
    m = CacheManager([GroupLayout("full"), GroupLayout("window", window=window, keep_first=keep)], page, [400, 400], 3)
    m.admit("a")
    n = 0
    for _ in range(rng.randrange(0, 40)):
        k = rng.randrange(1, 9)
        m.reserve({"a": k})
        m.commit("a", k)
        n += k
    m.reserve({"a": 30})                  # (taken for a step that has not been)
    m.fork("a", "b")
    assert m.n_tokens("b") == n and m.slot("b") != m.slot("a")
    for g in range(2):
        a, b = m.block_table("a", g), m.block_table("b", g)
        assert len(b) == -(-n // page) and [x < 0 for x in b] == [x < 0 for x in a[:len(b)]]
        assert not set(x for x in b if x >= 0) & set(a)
    m.check_invariants()
    with pytest.raises(CacheError):
        m.fork("a", "b")
    with pytest.raises(CacheError):
        m.fork("nobody", "c")
    assert not m.has("c")
    if all(p.n_free >= sum(x >= 0 for x in m.block_table("b", g)) for g, p in enumerate(m.pools)):
        m.fork("b", "c")
    else:
        with pytest.raises(OutOfPages):
            m.fork("b", "c")
        m.admit("c")
    with pytest.raises(OutOfPages):       # no slot
        m.fork("a", "d")
    for rid in "abc":
        m.release(rid)
    assert [p.n_free for p in m.pools] == [400, 400] and m.n_free_slots == 3
    m.check_invariants()


def test_a_fork_behind_a_window_needs_the_window_alone():
    """A long request whose layers all have a window holds few pages: a pool with exactly as many left takes its fork."""
    page, window = 4, 16
    m = CacheManager([GroupLayout("window", window=window)], page, [12], 2)
    m.admit("a")
    for _ in range(500):
        m.reserve({"a": 1})
        m.commit("a", 1)
    held = sum(p >= 0 for p in m.block_table("a", 0))
    assert held <= 6 and len(m.block_table("a", 0)) == 125
    m.fork("a", "b")
    assert m.pools[0].n_free == 12 - 2 * held
    m.release("b")
    m.admit("c")
    m.reserve({"c": page * (12 - 2 * held + 1)})
    m.release("a")
    m.check_invariants()


def test_a_fork_that_has_no_room_changes_nothing():
    m = CacheManager([GroupLayout("full"), GroupLayout("window", window=8)], 4, [10, 10], 3)
    m.admit("a")
    m.reserve({"a": 24})
    m.commit("a", 24)
    free = [p.n_free for p in m.pools]
    with pytest.raises(OutOfPages):
        m.fork("a", "b")
    assert not m.has("b") and [p.n_free for p in m.pools] == free and m.n_free_slots == 2
    m.check_invariants()


# ---- the end of a model's positions -------------------------------------------------------------------------------------
def test_a_wide_tree_at_the_end_of_the_positions(model_dirs, monkeypatch):
    """Two positions are left and nine tokens are drafted, none deeper than the second one; a third level is refused."""
    drafts_refs.install(monkeypatch)
    page, vocab, most = PAGE_SIZE["A"], CONFIG_A["vocab_size"], CONFIG_A["max_position_embeddings"]
    runner = make_runner(model_dirs["A"], page, n_pages=2 * most // page, max_requests=2)
    prompt = random_tokens(most - 2, vocab, seed=7)
    runner.admit(0)
    runner.step([StepEntry(0, prompt, [])])
    runner.admit(1)
    runner.step([StepEntry(1, [1, 2, 3], [])])
    tree = [-1, 0, 0, 0, -1, 4, 4, -1, 7]
    drafts = random_tokens(len(tree), vocab, seed=8)
    logits = runner.step_drafts([DraftEntry(1, [4] * 6, [-1, 0, 1, 2, 3, 4]), DraftEntry(0, drafts, tree)])
    for i in (3, 6, 8):
        assert rel_err(logits[6 + i], last_logits(model_dirs["A"], prompt + [drafts[tree[i]], drafts[i]])) < 1e-4
    runner.keep_drafts({0: [4, 6], 1: []})
    assert runner.n_tokens(0) == most
    with pytest.raises(BatchError, match="positions"):
        runner.step_drafts([DraftEntry(0, [1], [-1])])
    assert pages_held(runner, 0) == [most // page]
    runner.manager.check_invariants()


def test_a_tree_that_is_too_deep_is_refused(model_dirs, monkeypatch):
    drafts_refs.install(monkeypatch)
    page, most = PAGE_SIZE["A"], CONFIG_A["max_position_embeddings"]
    runner = make_runner(model_dirs["A"], page, n_pages=2 * most // page, max_requests=2)
    runner.admit(0)
    runner.step([StepEntry(0, [1] * (most - 2), [])])
    held = pages_held(runner, 0)
    with pytest.raises(BatchError, match="positions"):
        runner.step_drafts([DraftEntry(0, [1, 2, 3], [-1, 0, 1])])
    assert pages_held(runner, 0) == held
    runner.step_drafts([DraftEntry(0, [1, 2, 3], [-1, 0, 0])])


# ---- windows ------------------------------------------------------------------------------------------------------------
def windowed_runner(config, window, page, rt, seed=6):
    """A model whose second layer has a window and whose first two layers run twice."""
    spec, _ = spec_from_config(config)
    layers = list(spec.layers)
    layers[1] = layers[1].with_part("mixer", dataclasses.replace(layers[1].mixer, window=window))
    order = [0, 1, 0, 1] + list(range(2, len(layers)))
    spec = dataclasses.replace(spec, layers=tuple(layers), schedule=tuple(ScheduleEntry(layer=x, cache=i) for i, x in enumerate(order)))
    g = torch.Generator().manual_seed(seed)
    weights = {d.name: (1.0 + 0.1 * torch.randn(d.shape, generator=g) if len(d.shape) == 1 else
                        torch.randn(d.shape, generator=g) * d.shape[-1] ** -0.5).to(rt.dtype).to(rt.device) for d in declared_tensors(spec)}
    return ModelRunner(spec, weights, rt, page_size=page, n_pages=96, max_requests=4)


def check_windows(make, window, page, bound, n_prompt=70):
    """Trees behind contexts that windows have passed: every drafted token's logits are those of its path one token after another, the kept path
    goes on, and so does a fork behind it; a tree deeper than a window is refused."""
    runner, plain = make(), make()
    vocab = runner.spec.vocab_size
    assert runner.takes_drafts() and sorted(x.window or 0 for x in runner.storage.layouts) == [0, window]
    prompts = [random_tokens(n, vocab, seed=n) for n in (n_prompt, 3)]
    trees = [[-1, 0, 0, 1, -1, 4, 3, 6][:window + 4], [-1, 0, 1]]
    drafts = [random_tokens(len(t), vocab, seed=20 + i) for i, t in enumerate(trees)]
    for i, p in enumerate(prompts):
        runner.admit(i)
        runner.step([StepEntry(i, p, [])])
    if window <= 40:
        assert any(x < 0 for g, layout in enumerate(runner.storage.layouts) if layout.window for x in runner.manager.block_table(0, g))

    def one_by_one(tokens, n_wanted):
        plain.admit("p")
        plain.step([StepEntry("p", tokens[:-n_wanted], [])])
        rows = [plain.step([StepEntry("p", [t], [0])]).clone() for t in tokens[-n_wanted:]]
        plain.release("p")
        return torch.cat(rows)

    def path(tree, j):
        return (path(tree, tree[j]) if tree[j] >= 0 else []) + [j]

    logits = runner.step_drafts([DraftEntry(i, d, t) for i, (d, t) in enumerate(zip(drafts, trees))])
    at = 0
    for i, tree in enumerate(trees):
        for j in range(len(tree)):
            way = path(tree, j)
            want = one_by_one(prompts[i] + [drafts[i][k] for k in way], len(way))
            assert rel_err(logits[at + j].cpu(), want[-1].cpu()) < bound, (i, j)
        at += len(tree)
    runner.keep_drafts({0: path(trees[0], 6), 1: [0]})
    runner.fork(0, 2)
    held = {0: prompts[0] + [drafts[0][k] for k in path(trees[0], 6)], 1: prompts[1] + drafts[1][:1]}
    held[2] = list(held[0])
    chain = {0: [5, 6, 7], 1: [8, 9], 2: [1, 2, 3, 4]}
    got = runner.step_drafts([DraftEntry(r, c, list(range(-1, len(c) - 1))) for r, c in chain.items()])
    at = 0
    for r, c in chain.items():
        want = one_by_one(held[r] + c, len(c))
        assert rel_err(got[at:at + len(c)].cpu(), want.cpu()) < bound, r
        at += len(c)
    runner.keep_drafts({r: list(range(len(c))) for r, c in chain.items()})
    for r, c in chain.items():
        got = runner.step([StepEntry(r, [7], [0])])
        assert rel_err(got[0].cpu(), one_by_one(held[r] + c + [7], 1)[0].cpu()) < bound, r
    with pytest.raises(BatchError, match="window"):
        runner.step_drafts([DraftEntry(0, [1] * (window + 1), list(range(-1, window)))])
    runner.step_drafts([DraftEntry(0, [1] * window, list(range(-1, window - 1)))])
    runner.manager.check_invariants()


@pytest.mark.parametrize("window,page", [(24, 4), (17, 16), (5, 4)])
def test_trees_through_layers_with_windows(monkeypatch, window, page):
    drafts_refs.install(monkeypatch)
    rt = Runtime(torch.device("cpu"), torch.float32)
    check_windows(lambda: windowed_runner(CONFIG_A, window, page, rt), window, page, 1e-4)


# ---- everything in any order --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(6))
def test_steps_trees_forks_and_ends_in_any_order(model_dirs, monkeypatch, seed):
    """Requests that come, go on, draft, keep some of it or none, fork and end in random order: every row that is looked at has the logits of its
    request's tokens, and a request without drafts holds the pages of its tokens."""
    drafts_refs.install(monkeypatch)
    rng = random.Random(seed)
    page, vocab = PAGE_SIZE["A"], CONFIG_A["vocab_size"]
    runner = make_runner(model_dirs["A"], page, n_pages=40, max_requests=4)
    held, drafted, new = {}, {}, iter(range(10 ** 6))

    def some():
        return rng.sample(sorted(held), rng.randrange(1, len(held) + 1)) if held else []

    def path(rid):
        tokens, tree = drafted[rid]
        way, at = [], -1
        while True:
            children = [i for i, p in enumerate(tree) if p == at]
            if not children or rng.random() < 0.3:
                return way
            at = rng.choice(children)
            way.append(at)

    def look(logits, row, tokens):
        if rng.random() < 0.25:
            assert rel_err(logits[row], last_logits(model_dirs["A"], tokens)) < 1e-4

    for _ in range(120):
        what = rng.random()
        try:
            if what < 0.12 and runner.manager.n_free_slots:
                rid = next(new)
                runner.admit(rid)
                prompt = random_tokens(rng.randrange(1, 14), vocab, seed=rid)
                held[rid] = []
                logits = runner.step([StepEntry(rid, prompt, [len(prompt) - 1])])
                held[rid] = prompt
                look(logits, 0, prompt)
            elif what < 0.35 and held:
                entries = [StepEntry(r, random_tokens(rng.choice([1, 1, 1, 5]), vocab, seed=rng.randrange(10 ** 6)), [0]) for r in some()]
                logits = runner.step(entries)
                for i, e in enumerate(entries):
                    look(logits, i, held[e.rid] + list(e.tokens[:1]))
                    held[e.rid] = held[e.rid] + list(e.tokens)
                    drafted.pop(e.rid, None)
            elif what < 0.62 and held:
                entries = []
                for r in some():
                    n = rng.randrange(1, 11)
                    entries.append(DraftEntry(r, random_tokens(n, vocab, seed=rng.randrange(10 ** 6)), [rng.randrange(-1, i) for i in range(n)]))
                logits = runner.step_drafts(entries)
                row = 0
                for e in entries:
                    drafted[e.rid] = (list(e.tokens), list(e.parents))
                    for i in range(len(e.tokens)):
                        way, at = [], i
                        while at >= 0:
                            way, at = [e.tokens[at]] + way, e.parents[at]
                        look(logits, row, held[e.rid] + way)
                        row += 1
            elif what < 0.85 and drafted:
                kept = {r: path(r) for r in rng.sample(sorted(drafted), rng.randrange(1, len(drafted) + 1))}
                runner.keep_drafts(kept)
                for r, way in kept.items():
                    tokens = drafted.pop(r)[0]
                    held[r] = held[r] + [tokens[k] for k in way]
            elif what < 0.93 and held and runner.manager.n_free_slots:
                r, rid = rng.choice(sorted(held)), next(new)
                runner.fork(r, rid)
                held[rid] = list(held[r])
            elif held:
                r = rng.choice(sorted(held))
                runner.release(r)
                del held[r]
                drafted.pop(r, None)
        except OutOfPages:
            empty = [r for r in held if not held[r]]
            for r in empty or rng.sample(sorted(held), 1):
                runner.release(r)
                del held[r]
                drafted.pop(r, None)
        runner.manager.check_invariants()
        for r, tokens in held.items():
            assert runner.n_tokens(r) == len(tokens)
            if r not in drafted:
                assert pages_held(runner, r) == [-(-len(tokens) // page)]
    for r in list(held):
        runner.release(r)
    assert [p.n_free for p in runner.manager.pools] == [40]
