"""Drafted tokens, forks and log probabilities through the runner and the engine, against the plain implementation."""
import math

import pytest
import torch

import plain_qwen3
from helpers import CONFIG_A, CONFIG_B, CONFIG_C, CONFIG_D, PAGE_SIZE, random_tokens, rel_err
from inferrs_b200 import Engine, SamplingParams, kernels
from inferrs_b200.cache.manager import CacheError, OutOfPages
from inferrs_b200.engine.batch import BatchError, DraftEntry, StepEntry
from inferrs_b200.engine.loading import load_model_dir
from inferrs_b200.engine.runner import ModelRunner
from inferrs_b200.runtime import Runtime

pytestmark = pytest.mark.gpu

CONFIGS = {"A": CONFIG_A, "B": CONFIG_B, "C": CONFIG_C, "D": CONFIG_D}
# the bounds of the engine's other comparisons with the plain implementation (test_engine_gpu.py): the same sums in another order
TOL = {torch.float32: 1e-4, torch.bfloat16: 3e-2}


def make_runner(model_dir, dtype, page_size, n_pages=64, max_requests=4):
    rt = Runtime.cuda(dtype)
    spec, weights, _ = load_model_dir(model_dir, rt)
    return ModelRunner(spec, weights, rt, page_size=page_size, n_pages=n_pages, max_requests=max_requests)


def plain_logits(model_dir, tokens, dtype):
    cfg, w = plain_qwen3.read_model(model_dir)
    return plain_qwen3.forward(cfg, w, tokens, store=None if dtype == torch.float32 else dtype)


def path_of(parents, i):
    path = []
    while i >= 0:
        path.append(i)
        i = parents[i]
    return path[::-1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_a_tree_is_its_paths_one_by_one_and_what_is_kept_goes_on(model_dirs, name, dtype):
    vocab = CONFIGS[name]["vocab_size"]
    runner = make_runner(model_dirs[name], dtype, PAGE_SIZE[name])
    prompts = [random_tokens(19, vocab, seed=1), random_tokens(32, vocab, seed=2), random_tokens(1, vocab, seed=3)]
    trees = [[-1, 0, 0, 1, 1, 2, 3], [-1, 0, 1, 2], [-1, -1, 1]]
    drafts = [random_tokens(len(t), vocab, seed=10 + i) for i, t in enumerate(trees)]
    for i, p in enumerate(prompts):
        runner.admit(i)
        runner.step([StepEntry(i, p, [])])
    assert runner.takes_drafts()
    for again in range(2):        # a step whose tokens nobody keeps leaves no trace
        logits = runner.step_drafts([DraftEntry(i, d, t) for i, (d, t) in enumerate(zip(drafts, trees))])
        at = 0
        for i, (d, t) in enumerate(zip(drafts, trees)):
            for j in range(len(t)):
                tokens = prompts[i] + [d[k] for k in path_of(t, j)]
                assert rel_err(logits[at].cpu(), plain_logits(model_dirs[name], tokens, dtype)[-1]) < TOL[dtype], (again, i, j)
                at += 1
    kept = {0: path_of(trees[0], 6), 1: [0, 1], 2: path_of(trees[2], 2)}
    assert kept[0] == [0, 1, 3, 6] and kept[2] == [1, 2]
    runner.keep_drafts(kept)
    more = random_tokens(3, vocab, seed=50)
    for step, token in enumerate(more):
        got = runner.step([StepEntry(i, [token], [0]) for i in range(3)])
        for i in range(3):
            tokens = prompts[i] + [drafts[i][k] for k in kept[i]] + more[:step + 1]
            assert rel_err(got[i].cpu(), plain_logits(model_dirs[name], tokens, dtype)[-1]) < TOL[dtype], (step, i)
    assert kernels.attention_tree_error() == 0
    runner.manager.check_invariants()


def test_what_drafts_refuse(model_dirs):
    runner = make_runner(model_dirs["A"], torch.float32, PAGE_SIZE["A"], n_pages=8)
    runner.admit(0)
    runner.step([StepEntry(0, [1, 2, 3], [])])
    for bad in ([0], [-1, 1], [-1, -2]):
        with pytest.raises(BatchError):
            runner.step_drafts([DraftEntry(0, [5] * len(bad), bad)])
    with pytest.raises(BatchError):
        runner.step_drafts([DraftEntry(0, [5, 6], [-1])])
    with pytest.raises(BatchError):
        runner.keep_drafts({0: [0]})
    runner.step_drafts([DraftEntry(0, [5, 6, 7], [-1, 0, 0])])
    for bad in ([0, 3], [1, 0], [0, 0], [-1]):
        with pytest.raises(BatchError):
            runner.keep_drafts({0: bad})
    runner.keep_drafts({0: []})
    assert runner.n_tokens(0) == 3
    with pytest.raises(BatchError):
        runner.keep_drafts({0: [0]})
    runner.step_drafts([DraftEntry(0, [5], [-1])])
    runner.step([StepEntry(0, [9], [0])])         # wrote over them
    with pytest.raises(BatchError):
        runner.keep_drafts({0: [0]})


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["A", "D"])
def test_a_fork_goes_its_own_way(model_dirs, name, dtype):
    vocab = CONFIGS[name]["vocab_size"]
    runner = make_runner(model_dirs[name], dtype, PAGE_SIZE[name], n_pages=40, max_requests=3)
    prompt = random_tokens(2 * PAGE_SIZE[name] + 3, vocab, seed=4)
    runner.admit("a")
    runner.step([StepEntry("a", prompt, [])])
    runner.fork("a", "b")
    ways = {"a": random_tokens(6, vocab, seed=5), "b": random_tokens(6, vocab, seed=6)}
    for k in range(6):
        got = runner.step([StepEntry(r, [ways[r][k]], [0]) for r in "ab"])
        for i, r in enumerate("ab"):
            assert rel_err(got[i].cpu(), plain_logits(model_dirs[name], prompt + ways[r][:k + 1], dtype)[-1]) < TOL[dtype], (k, r)
    runner.fork("b", "c")
    got = runner.step([StepEntry("c", [1], [0])])
    assert rel_err(got[0].cpu(), plain_logits(model_dirs[name], prompt + ways["b"] + [1], dtype)[-1]) < TOL[dtype]
    runner.manager.check_invariants()
    free = [p.n_free for p in runner.manager.pools]
    with pytest.raises(OutOfPages):        # no slot
        runner.fork("a", "d")
    runner.release("c")
    runner.step([StepEntry("a", random_tokens(sum(free) * PAGE_SIZE[name] // 2 if name == "A" else 40, vocab, seed=8), [])])
    runner.manager.check_invariants()


def test_a_fork_without_room_changes_nothing(model_dirs):
    runner = make_runner(model_dirs["A"], torch.float32, PAGE_SIZE["A"], n_pages=5, max_requests=3)
    runner.admit("a")
    runner.step([StepEntry("a", [1] * (3 * PAGE_SIZE["A"]), [])])
    with pytest.raises(OutOfPages):
        runner.fork("a", "b")
    assert not runner.has("b") and runner.manager.pools[0].n_free == 2 and runner.manager.n_free_slots == 2
    runner.manager.check_invariants()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("overlap", [True, False])
def test_log_probabilities_of_generated_tokens(model_dirs, dtype, overlap):
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    vocab = CONFIG_B["vocab_size"]
    engine = Engine(model_dirs["B"], dtype=dtype, block_size=16, num_blocks=64, max_batch_size=4, max_tokens_per_step=32, overlap=overlap)
    prompts = [random_tokens(n, vocab, seed=n) for n in (9, 40, 3, 17)]
    options = [SamplingParams.greedy(max_tokens=6, logprobs=3), SamplingParams(max_tokens=5, seed=3, logprobs=0, ignore_eos=True),
               SamplingParams.greedy(max_tokens=7), SamplingParams(max_tokens=6, seed=4, logprobs=7, ignore_eos=True, repetition_penalty=1.5)]
    plain = engine.generate(prompts, [SamplingParams(**{**p.__dict__, "logprobs": None}) for p in options])
    done = engine.generate(prompts, options, return_requests=True)
    assert [r.output for r in done] == plain
    for r, p in zip(done, options):
        if p.logprobs is None:
            assert r.log_probs == []
            continue
        assert [x.token for x in r.log_probs] == r.output
        want = torch.log_softmax(plain_logits(model_dirs["B"], r.prompt + r.output, t).double(), -1)
        for k, x in enumerate(r.log_probs):
            row = want[len(r.prompt) + k - 1]
            # logits off by the engine's bound, relative to the largest one, move a log probability by twice that at most
            off = 4 * TOL[t] * float(plain_logits(model_dirs["B"], r.prompt + r.output, t).abs().max())
            assert abs(x.log_prob - float(row[x.token])) <= off
            assert abs(x.entropy + float((row.exp() * row).sum())) <= off * 4
            assert len(x.top) == p.logprobs and all(a[1] >= b[1] for a, b in zip(x.top, x.top[1:]))
            assert all(abs(lp - float(row[i])) <= off for i, lp in x.top)
            if p.is_greedy:
                assert x.top[0][0] == x.token and math.isclose(x.top[0][1], x.log_prob, rel_tol=0, abs_tol=1e-6)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompts_are_scored(model_dirs, dtype):
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    vocab = CONFIG_B["vocab_size"]
    engine = Engine(model_dirs["B"], dtype=dtype, block_size=16, num_blocks=64, max_batch_size=4, max_tokens_per_step=32)
    prompts = [random_tokens(n, vocab, seed=n) for n in (1, 2, 33, 65, 90)]
    for prompt, found in zip(prompts, engine.score(prompts, top=2)):
        assert [x.token for x in found] == prompt[1:]
        if len(prompt) == 1:
            continue
        logits = plain_logits(model_dirs["B"], prompt, t).double()
        want, off = torch.log_softmax(logits, -1), 4 * TOL[t] * float(logits.abs().max())
        for k, x in enumerate(found):
            assert abs(x.log_prob - float(want[k, x.token])) <= off and len(x.top) == 2
    assert engine.runner.manager.n_live == 0
    with pytest.raises(ValueError):
        engine.score(prompts, top=33)


def test_what_stays_is_a_path(model_dirs):
    runner = make_runner(model_dirs["A"], torch.float32, PAGE_SIZE["A"])
    runner.admit(0)
    runner.step([StepEntry(0, [1, 2, 3], [])])
    runner.step_drafts([DraftEntry(0, [5, 6, 7, 8], [-1, 0, 0, 1])])
    for bad in ([1], [0, 3], [0, 1, 2], [0, 2, 3], [0, 1, 3, 3]):
        with pytest.raises(BatchError):
            runner.keep_drafts({0: bad})
    runner.keep_drafts({0: [0, 1, 3]})
    assert runner.n_tokens(0) == 6
    with pytest.raises(BatchError):
        runner.step_drafts([])
    with pytest.raises(CacheError):
        runner.step_drafts([DraftEntry(0, [], [])])
    with pytest.raises(ValueError):
        runner.step_drafts([DraftEntry(0, [1], [-1]), DraftEntry(0, [2], [-1])])
    assert runner.n_tokens(0) == 6
    runner.manager.check_invariants()


@pytest.mark.parametrize("name", ["A", "D"])
def test_drafting_choosing_keeping_and_forking_give_the_greedy_tokens(model_dirs, name):
    """Trees whose tokens are half right, the model's choice among them, the path that it chose, and a fork that goes on alike: the
    tokens and log probabilities are those of one token after another."""
    vocab, n = CONFIGS[name]["vocab_size"], 14
    runner = make_runner(model_dirs[name], torch.float32, PAGE_SIZE[name])
    prompts = [random_tokens(11, vocab, seed=31), random_tokens(2 * PAGE_SIZE[name], vocab, seed=32)]
    greedy, wanted = [], []
    for prompt in prompts:
        tokens, log_probs = list(prompt), []
        for _ in range(n + 6):
            row = torch.log_softmax(plain_logits(model_dirs[name], tokens, torch.float32)[-1].double(), -1)
            tokens.append(int(row.argmax()))
            log_probs.append(float(row.max()))
        greedy.append(tokens[len(prompt):])
        wanted.append(log_probs)

    def choose(logits):
        rows = logits.shape[0]
        ids = torch.empty((rows, 1), dtype=torch.int32, device=logits.device)
        best = torch.empty((rows, 1), dtype=torch.float32, device=logits.device)
        given = torch.empty((rows, 1), dtype=torch.float32, device=logits.device)
        kernels.token_log_probs(logits, torch.zeros_like(ids), given, None, ids, best)
        return ids[:, 0].tolist(), best[:, 0].tolist()

    rids, out, scores = [0, 1], [[], []], [[], []]
    for r in rids:
        runner.admit(r)
    ids, best = choose(runner.step([StepEntry(r, prompts[r], [len(prompts[r]) - 1]) for r in rids]))
    for r in rids:
        out[r].append(ids[r])
        scores[r].append(best[r])
    turn = 0
    while min(map(len, out)) < n:
        if turn == 2:                  # a third request goes on from the second one, and the second one ends
            runner.fork(1, 2)
            runner.release(1)
            rids = [0, 2]
        entries = []
        for i, r in enumerate(rids):
            right = greedy[i][len(out[i]):] + [0] * 4
            wrong = (right[0] + 1) % vocab
            # the last token, a wrong one and the right one behind it, then two more right ones or (in turn) a wrong one
            entries.append(DraftEntry(r, [out[i][-1], wrong, right[0], wrong, right[1], right[2] if turn % 2 else wrong], [-1, 0, 0, 1, 2, 4]))
        ids, best = choose(runner.step_drafts(entries))
        kept = {}
        for i, r in enumerate(rids):
            e, at, path = entries[i], 6 * i, [0]
            while True:
                out[i].append(ids[at + path[-1]])
                scores[i].append(best[at + path[-1]])
                following = [k for k in range(6) if e.parents[k] == path[-1] and e.tokens[k] == out[i][-1]]
                if not following:
                    break
                path.append(following[0])
            kept[r] = path
            assert path[:3] == [0, 2, 4]
        runner.keep_drafts(kept)
        turn += 1
    assert turn >= 3
    for i in range(2):
        assert out[i][:n] == greedy[i][:n]
        # logits off by the engine's bound, relative to the largest one, move a log probability by twice that at most
        off = 2 * TOL[torch.float32] * float(plain_logits(model_dirs[name], prompts[i] + greedy[i], torch.float32).abs().max())
        assert all(abs(a - b) <= off for a, b in zip(scores[i][:n], wanted[i]))
    runner.manager.check_invariants()
