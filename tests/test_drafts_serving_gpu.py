"""Log probabilities while requests are preempted, stopped and aborted, and scores of prompts beside live requests."""
from __future__ import annotations

import pytest
import torch

from helpers import CONFIG_B, random_tokens
from inferrs_b200 import Engine, SamplingParams
from test_drafts_engine_gpu import TOL, plain_logits

pytestmark = pytest.mark.gpu


def options(i, **more):
    return SamplingParams(max_tokens=24, seed=4 + i, temperature=0.8, top_k=0, top_p=1.0, repetition_penalty=1.0 + 0.2 * (i % 2), **more)


@pytest.mark.parametrize("overlap", [True, False])
def test_preempted_requests_record_every_token_once(model_dirs, overlap):
    """A request that is computed again keeps what was recorded of its tokens; each has one record, of the distribution behind the tokens ahead."""
    prompts = [random_tokens(n, CONFIG_B["vocab_size"], seed=80 + n) for n in (1, 9, 40, 100)]
    kw = dict(dtype="f32", block_size=16, num_blocks=13, max_batch_size=4, max_tokens_per_step=12, prefill_chunk=7, overlap=overlap)
    want = Engine(model_dirs["B"], **kw).generate(prompts, [options(i, ignore_eos=i != 3) for i in range(4)])
    eng = Engine(model_dirs["B"], **kw)
    done = eng.generate(prompts, [options(i, logprobs=(0, 5, None, 2)[i], ignore_eos=i != 3) for i in range(4)], return_requests=True)
    assert eng.stats()["preemptions"] > 0 and [r.output for r in done] == want
    for r, n in zip(done, (0, 5, None, 2)):
        if n is None:
            assert r.log_probs == []
            continue
        assert [x.token for x in r.log_probs] == r.output and all(len(x.top) == n for x in r.log_probs)
        logits = plain_logits(model_dirs["B"], r.prompt + r.output, torch.float32)
        rows, off = torch.log_softmax(logits.double(), -1), 2 * TOL[torch.float32] * float(logits.abs().max())
        for k, x in enumerate(r.log_probs):
            assert abs(x.log_prob - float(rows[len(r.prompt) + k - 1, x.token])) <= off


@pytest.mark.parametrize("overlap", [True, False])
def test_scores_beside_live_requests(model_dirs, overlap):
    """Prompts are scored between the steps of live requests, one of which is aborted: nobody's tokens or records change."""
    vocab = CONFIG_B["vocab_size"]
    kw = dict(dtype="f32", block_size=16, num_blocks=64, max_batch_size=4, max_tokens_per_step=24, overlap=overlap)
    prompts = [random_tokens(n, vocab, seed=n) for n in (5, 33, 18)]
    scored = [random_tokens(n, vocab, seed=50 + n) for n in (30, 2, 25)]
    alone = Engine(model_dirs["B"], **kw)
    want = alone.generate(prompts, [options(i, logprobs=3) for i in range(3)], return_requests=True)
    want_scores = alone.score(scored, top=4)
    eng = Engine(model_dirs["B"], **kw)
    rids = [eng.add_request(p, options(i, logprobs=3)) for i, p in enumerate(prompts)]
    # each side's logits are off by the engine's bound, relative to the largest one, which moves a log probability by twice that at most
    off = 4 * TOL[torch.float32] * max(float(plain_logits(model_dirs["B"], r.prompt + r.output, torch.float32).abs().max()) for r in want)
    done, turn = {}, 0
    while eng.has_work():
        for r in eng.step():
            done[r.rid] = r
        if turn % 5 == 2:
            for a, b in zip(eng.score(scored, top=4), want_scores):
                assert [x.token for x in a] == [x.token for x in b]
                assert all(abs(x.log_prob - y.log_prob) <= off for x, y in zip(a, b))
        if turn == 8:
            aborted = eng.abort(rids[2])
            done[rids[2]] = aborted
        turn += 1
    assert [done[r].output for r in rids[:2]] == [r.output for r in want[:2]]
    for r, w in zip((done[r] for r in rids), want):
        assert [x.token for x in r.log_probs] == r.output == w.output[:len(r.output)]
        assert all(abs(x.log_prob - y.log_prob) <= off for x, y in zip(r.log_probs, w.log_probs))
    assert done[rids[2]].finish_reason == "cancelled" and eng.runner.manager.n_live == 0
    eng.runner.manager.check_invariants()
