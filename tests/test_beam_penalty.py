"""Length penalties of beam search, up to the largest that hypotheses can be ranked with, and beyond."""
import math

import pytest

import beam_models
import plain_beam
from pico_vllm_b200.errors import ConfigError
from test_beam_search import on_cpu  # noqa: F401  (a fixture)


@pytest.mark.parametrize("tokens,penalty", [(11, 300.0), (11, 252.4), (2, 873.5), pytest.param(2, 10 ** 400, id="whole"), (16, 1e308), (4096, 72.8), (3, 1e30)])
def test_penalties_that_nothing_can_be_ranked_with_are_refused(tokens, penalty):
    """Their powers are no float64, or what is divided by them would lose digits."""
    from pico_vllm_b200 import BeamParams
    with pytest.raises(ConfigError, match="length_penalty"):
        BeamParams(max_new_tokens=tokens, length_penalty=penalty)


@pytest.mark.parametrize("tokens,penalty", [(1, 1e300), pytest.param(1, 10 ** 400, id="whole"), (2, 873.0), (2, 873), (11, 252.3), (4096, 72.75), (16, 218.25)])
def test_the_largest_penalties(tokens, penalty):
    """The smallest and the largest sums of log-probabilities that there are have values apart."""
    from pico_vllm_b200 import BeamParams
    from pico_vllm_b200.engine import BeamSearch
    params = BeamParams(max_new_tokens=tokens, length_penalty=penalty)

    class search:
        _value, params = BeamSearch._value, None
    search.params = params
    for score in (-2.0 ** -149, -1.0, -3.4e38):
        a, b = (BeamSearch._value(search, s, tokens) for s in (score * (1 + 2.0 ** -23), score))
        assert -math.inf < a < b <= -2.0 ** -1022


@pytest.mark.parametrize("penalty", [20.0, 290.0])
def test_a_search_with_a_large_penalty(on_cpu, penalty):  # noqa: F811
    from pico_vllm_b200 import BeamParams
    name, beams, tokens = "qwen2/b", 3, 8
    prompts = beam_models.prompts_of(name, (8, 5))
    next_logits = beam_models.model(name)[3]
    end = plain_beam.search(next_logits, prompts[0], beams, tokens, None, 1.0)[0][0][2][3]
    llm = beam_models.llm(name, "cpu", beams, end_token=end)
    params = BeamParams(beams=beams, max_new_tokens=tokens, length_penalty=penalty)
    outs = llm.beam_search(prompts, params)
    assert any(h.finish_reason == "eos" for o in outs for h in o.hypotheses)
    assert all(h.value == h.score / len(h.token_ids) ** penalty for o in outs for h in o.hypotheses)
    assert all([h.value for h in o.hypotheses] == sorted((h.value for h in o.hypotheses), reverse=True) for o in outs)
    llm.cache.check()
