"""Beam search through the whole engine on the GPU: the operators together, as they are used, against a plain search in float64."""
import math

import pytest
import torch

import beam_models
from test_beam_search import _Told, _manager, compare

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("name,lengths,beams,tokens,penalty", beam_models.SEARCHES)
@pytest.mark.parametrize("graphs", [False, True])
def test_search_equals_plain(name, lengths, beams, tokens, penalty, graphs):
    import plain_beam
    from pico_vllm_b200 import BeamParams
    prompts = beam_models.prompts_of(name, lengths)
    next_logits = beam_models.model(name)[3]
    end = None
    if graphs:              # (half of the cases with an end token)
        end = plain_beam.search(next_logits, prompts[0], beams, tokens, None, penalty)[0][0][2][min(3, tokens - 1)]
    llm = beam_models.llm(name, DEV, beams, end_token=end, use_cuda_graph=graphs)
    params = BeamParams(beams=beams, max_new_tokens=tokens, length_penalty=penalty)
    outs = llm.beam_search(prompts, params)
    compare(outs, prompts, next_logits, beams, tokens, end, penalty, 2e-5)
    assert llm.beam_search(prompts, params) == outs
    llm.cache.check()
    assert all(g.pool.in_use == 0 for g in llm.cache.groups)


@pytest.mark.parametrize("name,beams", [("qwen2/d", 4), ("qwen2/e", 8), ("recurrent/a", 4)])
def test_scores_are_those_of_the_tokens_in_bfloat16(name, beams):
    """Each hypothesis run again as a request of its own, token by token, has the score that the search gave it: no beam read another's keys, values or
    states.  (In 16 bits products of other batch sizes differ, each logit by some 1e-2 of the largest.)"""
    from pico_vllm_b200 import BeamParams
    from pico_vllm_b200.engine import StepItem
    prompts = beam_models.prompts_of(name, (50, 3, 33))
    llm = beam_models.llm(name, DEV, beams, at_once=3, dtype="bfloat16", use_cuda_graph=True, max_num_batched_tokens=64, max_cache_tokens=4096)
    outs = llm.beam_search(prompts, BeamParams(beams=beams, max_new_tokens=24, ignore_eos=True))
    for p, o in zip(prompts, outs):
        assert len({tuple(h.token_ids) for h in o.hypotheses}) == beams
        for h in o.hypotheses[:3]:
            slot = llm.cache.acquire("again")
            total, most = 0.0, 0.0
            logits = llm.runner.step([StepItem(slot, p, (len(p) - 1,))])
            for k, t in enumerate(h.token_ids):
                lp = logits[0].double().log_softmax(0)
                total, most = total + float(lp[t]), max(most, float(logits[0].abs().max()))
                if k + 1 < len(h.token_ids):
                    logits = llm.runner.step([StepItem(slot, [t], (0,))])
            llm.cache.release(slot)
            assert abs(total - h.score) <= 2e-2 * most * math.sqrt(len(h.token_ids)), (total, h.score, most)


DESIGNS = [(m, k) for m, names in (("zapipel", "pqmr"), ("zikupel", "abcd"), ("zazilix", "abcd"), ("banazen", "abc"), ("vanapel", "abcd"), ("zegorax", "abcd"))
           for k in names]


@pytest.mark.parametrize("design,name", DESIGNS)
def test_every_design_searches(design, name):
    """Latents, pages of windows, states of every kind, layers that read another's cache: each hypothesis run again as a request of its own has the score
    that the search gave it, in 32 bits.  A logit is off by at most 5e-5 of the largest (the designs' own tests), a token's log-probability by twice that; what
    a beam would take from another one is off by 1e-2 and more."""
    import importlib
    from pico_vllm_b200 import BeamParams
    from pico_vllm_b200.engine import StepItem
    from pico_vllm_b200.registry import config_from_dict
    module = importlib.import_module(f"test_{design}_gpu")
    raw = module.SHAPES[name]
    tensors = module._tensors(name) if design == "zapipel" else module._tensors(raw, module.SEEDS[name])
    llm = beam_models.llm_of(config_from_dict(raw), tensors, DEV, 4, page_size=8, use_cuda_graph=True, max_num_batched_tokens=24, max_model_len=64,
                             max_cache_tokens=640)
    import helpers
    prompts = [helpers.random_ids(n, llm.model.vocab_size, 60 + n) for n in (27, 8)]
    moved, reorder = [], llm.cache.reorder
    llm.cache.reorder = lambda slots, parents, *more: (moved.extend(q != p for f in parents for p, q in enumerate(f)), reorder(slots, parents, *more))[1]
    outs = llm.beam_search(prompts, BeamParams(beams=4, max_new_tokens=21, ignore_eos=True))
    assert sum(moved) >= 4                  # beams died and others branched off
    for p, o in zip(prompts, outs):
        assert len({tuple(h.token_ids) for h in o.hypotheses}) == 4
        for h in o.hypotheses:
            slot = llm.cache.acquire("again")
            logits = llm.runner.step([StepItem(slot, p, (len(p) - 1,))])
            total, most = 0.0, 0.0
            for k, t in enumerate(h.token_ids):
                total, most = total + float(logits[0].double().log_softmax(0)[t]), max(most, float(logits[0].abs().max()))
                if k + 1 < len(h.token_ids):
                    logits = llm.runner.step([StepItem(slot, [t], (0,))])
            llm.cache.release(slot)
            assert abs(total - h.score) <= 1e-4 * most * len(h.token_ids), (total, h.score, most)
    llm.cache.check()


def test_branches_on_the_device():
    """The cache's branches with the kernels: fork, reorder (with the indices here or on the device), compact, and pages of a window."""
    import random
    rng = random.Random(11)
    from pico_vllm_b200.cache import CacheManager
    like = _manager()
    m = CacheManager([g.spec for g in (like.groups[0], like.groups[1], like.groups[0])] + list(like.state_specs.values()), 4, 60, 8, 80, torch.float32, DEV,
                     poison_freed=True)
    told = _Told(m)
    a, b = m.acquire("a"), m.acquire("b")
    told.write(a, 11)
    told.write(b, 6)
    fa, fb = [a] + m.fork(a, 3), [b] + m.fork(b, 2)
    for f in (fa, fb):
        for s in f[1:]:
            told.text[s] = list(told.text[f[0]])
    for step in range(14):
        for s in fa + fb:
            told.write(s, 1)
        some = [fa, fb]
        parents = [[rng.randrange(len(f)) for _ in f] for f in some]
        texts = {s: told.text[f[q]] for f, p in zip(some, parents) for s, q in zip(f, p)}
        if step % 2:
            m.reorder(some, parents)
        else:
            for f, p in zip(some, parents):
                m.reorder([f], [p], (torch.tensor([f], dtype=torch.int32, device=DEV), torch.tensor([p], dtype=torch.int32, device=DEV)))
        told.text.update({s: list(t) for s, t in texts.items()})
        if step == 9:
            m.release(fa[0])
            del told.text[fa[0]]
            fa = fa[1:]
            assert m.compact() > 0
        told.check()


def test_command_line_searches(tmp_path, capsys):
    import helpers
    from pico_vllm_b200 import LLM, BeamParams
    from pico_vllm_b200.cli import main
    helpers.write_tiny_model("a", tmp_path, dtype="float32")
    rc = main(["run", "--model", str(tmp_path), "--dtype", "float32", "--prompt-ids", "5,17,3", "--prompt-ids", "9", "--max-new-tokens", "5", "--beams", "3",
               "--length-penalty", "0.5", "--num-gpu-blocks", "32", "--ignore-eos"])
    assert rc == 0
    lines = [line for line in capsys.readouterr().out.splitlines() if line.startswith("[")]
    llm = LLM(str(tmp_path), dtype="float32", num_pages=32, max_num_seqs=3)
    outs = llm.beam_search([[5, 17, 3], [9]], BeamParams(beams=3, max_new_tokens=5, length_penalty=0.5, ignore_eos=True))
    assert lines == [f"[{i}] {h.score:.6f} {' '.join(map(str, h.token_ids))}" for i, o in enumerate(outs) for h in o.hypotheses]


@pytest.mark.parametrize("ahead", [True, False])
def test_pages_brought_together_between_steps_change_no_token(ahead):
    """Also with a step in flight and steps that are replayed: a long request goes on while short ones end below it."""
    from pico_vllm_b200 import SamplingParams
    prompts = beam_models.prompts_of("qwen2/b", (30, 41, 7, 25))
    lengths = (3, 40, 5, 24)
    llm = beam_models.llm("qwen2/b", DEV, 4, at_once=1, use_cuda_graph=True, async_scheduling=ahead)
    want = [llm.generate([p], SamplingParams(temperature=0.0, max_new_tokens=n, ignore_eos=True))[0].token_ids for p, n in zip(prompts, lengths)]
    ids = [llm.submit(p, max_new_tokens=n, temperature=0.0, ignore_eos=True) for p, n in zip(prompts, lengths)]
    llm.mark_finished()
    done, copied = {}, 0
    while not llm.is_done():
        done.update(llm.step())
        copied += llm.compact_cache()
        llm.cache.check()
    assert copied > 0 and [done[i] for i in ids] == [p + w for p, w in zip(prompts, want)]
