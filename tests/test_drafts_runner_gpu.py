"""Drafted tokens and forks beside replayed steps."""
from __future__ import annotations

import pytest
import torch

from helpers import CONFIG_A, CONFIG_B, CONFIG_C, CONFIG_D, PAGE_SIZE, random_tokens, rel_err
from inferrs_b200 import kernels
from inferrs_b200.engine.batch import DraftEntry, StepEntry
from inferrs_b200.engine.loading import load_model_dir
from inferrs_b200.engine.runner import ModelRunner
from inferrs_b200.runtime import Runtime
from test_drafts_engine_gpu import TOL, plain_logits
from test_drafts_runner import check_windows, windowed_runner

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keep", [True, False])
def test_replayed_steps_behind_a_tree_that_reached_beyond_their_tables(model_dirs, dtype, keep):
    """The block tables of replayed steps end with the longest context that the runner was told; a tree may be wider than what is left of it."""
    page, vocab = PAGE_SIZE["A"], CONFIG_A["vocab_size"]
    rt = Runtime.cuda(dtype)
    spec, weights, _ = load_model_dir(model_dirs["A"], rt)
    runner = ModelRunner(spec, weights, rt, page_size=page, n_pages=32, max_requests=2, max_context=3 * page)
    assert runner.graphs is not None and runner.graphs.fixed_pages == [3]
    prompt = random_tokens(3 * page - 3, vocab, seed=1)
    runner.admit(0)
    runner.step([StepEntry(0, prompt, [])])
    drafts = random_tokens(2 * page, vocab, seed=2)
    logits = runner.step_drafts([DraftEntry(0, drafts, [-1] + [0] * (2 * page - 1))])
    assert rel_err(logits[-1].cpu(), plain_logits(model_dirs["A"], prompt + [drafts[0], drafts[-1]], dtype)[-1]) < TOL[dtype]
    tokens = list(prompt)
    if keep:
        runner.keep_drafts({0: [0]})
        tokens.append(drafts[0])
    for token in (3, 4):
        tokens.append(token)
        got = runner.step([StepEntry(0, [token], [0])])
        assert rel_err(got[0].cpu(), plain_logits(model_dirs["A"], tokens, dtype)[-1]) < TOL[dtype]
    assert runner.graphs.captured and runner.n_tokens(0) == len(tokens)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_wide_tree_at_the_end_of_the_positions(model_dirs, dtype):
    page, vocab, most = PAGE_SIZE["A"], CONFIG_A["vocab_size"], CONFIG_A["max_position_embeddings"]
    rt = Runtime.cuda(dtype)
    spec, weights, _ = load_model_dir(model_dirs["A"], rt)
    runner = ModelRunner(spec, weights, rt, page_size=page, n_pages=most // page + 8, max_requests=2)
    prompt = random_tokens(most - 3, vocab, seed=7)
    runner.admit(0)
    runner.step([StepEntry(0, prompt, [])])
    tree = [-1] + [0] * 20
    drafts = random_tokens(len(tree), vocab, seed=8)
    logits = runner.step_drafts([DraftEntry(0, drafts, tree)])
    for i in (0, 1, 20):
        tokens = prompt + drafts[:1] + ([drafts[i]] if i else [])
        assert rel_err(logits[i].cpu(), plain_logits(model_dirs["A"], tokens, dtype)[-1]) < TOL[dtype]
    runner.keep_drafts({0: [0, 20]})
    got = runner.step([StepEntry(0, [9], [0])])
    assert rel_err(got[0].cpu(), plain_logits(model_dirs["A"], prompt + [drafts[0], drafts[20], 9], dtype)[-1]) < TOL[dtype]
    assert runner.n_tokens(0) == most


@pytest.mark.parametrize("config,window,n_prompt", [(CONFIG_B, 24, 70), (CONFIG_C, 17, 90), (CONFIG_D, 24, 70), (CONFIG_D, 130, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_trees_through_layers_with_windows(config, window, n_prompt, dtype):
    rt = Runtime.cuda(dtype)
    check_windows(lambda: windowed_runner(config, window, 16, rt), window, 16, TOL[dtype], n_prompt)
    assert kernels.attention_tree_error() == 0
