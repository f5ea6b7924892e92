"""Beam search on the GPU over models whose next token hangs on the whole context: a beam that read another one's keys, values or states would be seen,
and searches that leave out what has to move are."""
import math

import pytest
import torch

import context_models
import plain_beam
from test_beam_search import compare

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("name,lengths,beams,tokens,penalty", context_models.SEARCHES)
@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("ends", [False, True])
def test_search_equals_plain(monkeypatch, name, lengths, beams, tokens, penalty, ends, graphs):
    from pico_vllm_b200 import BeamParams
    prompts, next_logits = context_models.prompts_of(name, lengths), context_models.model(name)[3]
    end = plain_beam.search(next_logits, prompts[0], beams, tokens, None, penalty)[0][0][2][3] if ends else None
    params = BeamParams(beams=beams, max_new_tokens=tokens, length_penalty=penalty)
    llm = context_models.llm(name, DEV, beams, end_token=end, use_cuda_graph=graphs)
    moved = context_models.moves(llm)
    outs = llm.beam_search(prompts, params)
    compare(outs, prompts, next_logits, beams, tokens, end, penalty, context_models.OFF)
    assert moved[0] > 0 and llm.beam_search(prompts, params) == outs
    llm.cache.check()
    if not ends:
        for what in ("copies", "reorder"):
            # (an engine of its own: the pages and states of one that has searched hold what would have been copied)
            other = context_models.llm(name, DEV, beams, use_cuda_graph=graphs)
            with monkeypatch.context() as m:
                context_models.leave_out(m, other, what)
                assert all(context_models.apart(outs, other.beam_search(prompts, params))), what


def again(llm, prompt, hypothesis):
    """The sum of the hypothesis' log-probabilities as a request of its own, token by token, and the largest logit on the way."""
    from pico_vllm_b200.engine import StepItem
    slot = llm.cache.acquire("again")
    logits = llm.runner.step([StepItem(slot, prompt, (len(prompt) - 1,))])
    total, most = 0.0, 0.0
    for k, t in enumerate(hypothesis.token_ids):
        total, most = total + float(logits[0].double().log_softmax(0)[t]), max(most, float(logits[0].abs().max()))
        if k + 1 < len(hypothesis.token_ids):
            logits = llm.runner.step([StepItem(slot, [t], (0,))])
    llm.cache.release(slot)
    return total, most


# What of the largest logit a token's log-probability may be off by between two batches in 16 bits.  The sums are in 32 bits in both, in another order; a stored
# value differs where its sum lies next to a border of rounding, by one step of 2^-7, otherwise not at all.  The model's ten stored values on the way of a token
# through a layer (norm, products, scores' weights, outputs), were one in eight of each to differ, would move a logit by 2^-7 * sqrt(10 * layers / 8) of the
# logits' spread, a third of the largest: 2^-7 / 3 * sqrt(30 / 8) = 5e-3 with three layers.  Tokens' errors are of either sign.
STEP = 5e-3


@pytest.mark.parametrize("name,beams", [("untied/d", 4), ("untied/e", 8), ("qwen2/b", 3), ("whole/a", 4), ("whole/c", 3), ("whole/d", 3)])
def test_scores_are_those_of_the_tokens_in_bfloat16(monkeypatch, name, beams):
    """Each hypothesis run again by itself has the score that the search gave it; hypotheses of searches that leave out what has to move have not."""
    from pico_vllm_b200 import BeamParams
    prompts = context_models.prompts_of(name, (50, 3, 33))
    options = dict(at_once=3, dtype="bfloat16", use_cuda_graph=True, max_num_batched_tokens=64, max_cache_tokens=4096)
    llm = context_models.llm(name, DEV, beams, **options)
    params = BeamParams(beams=beams, max_new_tokens=24, ignore_eos=True)
    moved = context_models.moves(llm)

    def worst(outs):
        """For each prompt: by how many times what is allowed the worst score is off."""
        seen = []
        for p, o in zip(prompts, outs):
            off = [(abs(total - h.score), most, len(h.token_ids)) for h in o.hypotheses for total, most in [again(llm, p, h)]]
            seen.append(max(d / (STEP * most * math.sqrt(n)) for d, most, n in off))
        return seen
    outs = llm.beam_search(prompts, params)
    assert moved[0] > 0 and all(len({tuple(h.token_ids) for h in o.hypotheses}) == beams for o in outs)
    right = worst(outs)
    print(name, "scores off by, of what is allowed:", [round(v, 4) for v in right])
    assert max(right) <= 1, right
    for what in ("copies", "reorder"):
        other = context_models.llm(name, DEV, beams, **options)
        with monkeypatch.context() as m:
            context_models.leave_out(m, other, what)
            outs = other.beam_search(prompts, params)
        wrong = worst(outs)
        print(name, what, "left out:", [round(v, 2) for v in wrong])
        assert max(wrong) > 2, (what, wrong)
