"""Beam search on the CPU, with the kernels replaced by torch doubles, over models whose next token hangs on the whole context: a search that leaves out what
has to move ends elsewhere, and so do requests whose pages are brought together without being copied."""
import pytest

import context_models
import plain_beam
from test_beam_search import compare, on_cpu  # noqa: F401  (a fixture)


@pytest.mark.parametrize("name", sorted({s[0] for s in context_models.SEARCHES}))
def test_the_next_token_hangs_on_the_whole_context(name):
    """Another token anywhere before moves the logits by far more than what they may be off by."""
    ids = context_models.prompts_of(name, (12,))[0]
    next_logits, vocab = context_models.model(name)[3], context_models.vocab(name)
    before = next_logits(ids)
    for at in range(len(ids)):
        other = ids[:at] + [(ids[at] + 7) % vocab] + ids[at + 1:]
        assert (next_logits(other) - before).abs().max() > 1e4 * context_models.OFF
    assert before.abs().max() < 60


@pytest.mark.parametrize("name,lengths,beams,tokens,penalty", context_models.SEARCHES)
def test_searches_that_leave_out_what_has_to_move_end_elsewhere(on_cpu, monkeypatch, name, lengths, beams, tokens, penalty):  # noqa: F811
    from pico_vllm_b200 import BeamParams
    prompts, next_logits = context_models.prompts_of(name, lengths), context_models.model(name)[3]
    params = BeamParams(beams=beams, max_new_tokens=tokens, length_penalty=penalty)
    llm = context_models.llm(name, "cpu", beams)
    moved = context_models.moves(llm)
    outs = llm.beam_search(prompts, params)
    compare(outs, prompts, next_logits, beams, tokens, None, penalty, context_models.OFF)
    assert moved[0] > 0 and all(len(set(o.hypotheses[0].token_ids)) > 1 for o in outs)
    for what in ("copies", "states", "reorder")[::1 if name.startswith("recurrent") else 2]:
        other = context_models.llm(name, "cpu", beams)
        with monkeypatch.context() as m:
            context_models.leave_out(m, other, what)
            assert all(context_models.apart(outs, other.beam_search(prompts, params))), what


@pytest.mark.parametrize("name,lengths,beams,tokens,penalty", context_models.SEARCHES[0:6:3] + context_models.SEARCHES[5:6])
def test_search_with_an_end_token(on_cpu, name, lengths, beams, tokens, penalty):  # noqa: F811
    from pico_vllm_b200 import BeamParams
    prompts, next_logits = context_models.prompts_of(name, lengths), context_models.model(name)[3]
    end = plain_beam.search(next_logits, prompts[0], beams, tokens, None, penalty)[0][0][2][3]
    llm = context_models.llm(name, "cpu", beams, end_token=end)
    outs = llm.beam_search(prompts, BeamParams(beams=beams, max_new_tokens=tokens, length_penalty=penalty))
    compare(outs, prompts, next_logits, beams, tokens, end, penalty, context_models.OFF)
    assert any(h.finish_reason == "eos" for o in outs for h in o.hypotheses)


@pytest.mark.parametrize("left_out", [False, True])
def test_pages_brought_together(on_cpu, monkeypatch, left_out):  # noqa: F811
    """A request goes on while others below it end; its tokens are those of a request alone only if its pages are copied."""
    from pico_vllm_b200 import SamplingParams
    prompts, lengths = context_models.prompts_of("untied/a", (21, 40, 18)), (2, 14, 5)
    llm = context_models.llm("untied/a", "cpu", 3, at_once=1)
    want = [llm.generate([p], SamplingParams(temperature=0.0, max_new_tokens=n, ignore_eos=True))[0].token_ids for p, n in zip(prompts, lengths)]
    if left_out:
        context_models.leave_out(monkeypatch, llm, "copies")
    ids = [llm.submit(p, max_new_tokens=n, temperature=0.0, ignore_eos=True) for p, n in zip(prompts, lengths)]
    llm.mark_finished()
    done, copied = {}, 0
    while not llm.is_done():
        done.update(llm.step())
        copied += llm.compact_cache()
        llm.cache.check()
    assert copied > 0 and (done[ids[1]] == prompts[1] + want[1]) != left_out
    assert done[ids[0]] == prompts[0] + want[0]
