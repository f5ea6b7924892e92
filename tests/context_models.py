"""Models whose next token hangs on the whole context, so that a beam that reads another one's keys, values or states goes another way: the small
models of helpers.py with a head of their own (a tied, scaled table is mostly the last token's own row), and those with states."""
import torch

import beam_models
import helpers
import plain_qwen2

OFF = 2e-5          # what a logit of the 32-bit path may be off by (the largest logits are below 60 here)


def untied(name):
    from pico_vllm_b200.registry import config_from_dict
    from pico_vllm_b200.weights import random_tensors
    cfg = config_from_dict(dict(helpers.TINY[name]["raw"], tie_word_embeddings=False))
    tensors = random_tensors(cfg, helpers.TINY[name]["seed"], dtype=torch.float32)
    tensors["lm_head.weight"] = tensors["lm_head.weight"] * 12
    pcfg = helpers.plain_config(cfg)
    double = {k: v.double() for k, v in tensors.items()}
    return cfg, tensors, helpers.TINY[name]["page_size"], lambda ids: plain_qwen2.forward(torch.tensor(ids), double, pcfg, torch.float64)[-1]


def whole(name):
    """A model with states whose tokens all go to all experts: in 16 bits a choice of experts hangs on the last bit."""
    import plain_zazilix
    import test_zazilix_gpu as zazilix
    from pico_vllm_b200.registry import config_from_dict
    raw = zazilix._raw(name, "bfloat16")
    tensors = zazilix._tensors(raw, zazilix.SEEDS[name])
    tensors["head"] = tensors["head"] * 12
    return config_from_dict(raw), tensors, 8, lambda ids: plain_zazilix.forward(raw, tensors, ids)[-1]


def model(name):
    """(config, tensors, page size, next_logits in float64)"""
    family, which = name.split("/")
    return {"untied": untied, "whole": whole}[family](which) if family in ("untied", "whole") else beam_models.model(name)


def vocab(name):
    cfg = model(name)[0]
    return cfg.vocab_size if hasattr(cfg, "vocab_size") else cfg.vocab


def prompts_of(name, lengths):
    return [helpers.random_ids(n, vocab(name), 700 + n) for n in lengths]


def llm(name, device, beams, at_once=2, end_token=None, dtype="float32", **options):
    config, tensors, page, _ = model(name)
    return beam_models.llm_of(config, tensors, device, beams, at_once, end_token, dtype, **{"page_size": page, **options})


# (model, prompts' lengths, beams, tokens, length penalty): pages that are partly filled, full and fresh; windows; states
SEARCHES = [("untied/a", (5, 16, 37), 4, 12, 1.0), ("untied/c", (11, 5), 8, 8, 2.0), ("untied/d", (20, 47), 3, 10, 0.5), ("untied/e", (31, 6), 5, 9, 1.0),
            ("qwen2/b", (8, 30), 3, 14, 0.0), ("recurrent/a", (7, 16), 4, 10, 1.0), ("recurrent/b", (10, 8), 3, 10, 0.5)]


def moves(llm):
    """Counts what the cache's reorder is asked to move, from now on."""
    count, reorder = [0], llm.cache.reorder

    def counted(slots, parents, *more):
        count[0] += sum(q != p for f in parents for p, q in enumerate(f))
        return reorder(slots, parents, *more)
    llm.cache.reorder = counted
    return count


def leave_out(monkeypatch, llm, what):
    """The search goes on without a part of what it has to move: pages (and states that are copied where a request branches), states, or all of a reorder."""
    import pico_vllm_b200.ops as ops
    if what == "copies":
        monkeypatch.setattr(ops, "copy_pages", lambda tensors, src, dst: tensors)
    elif what == "states":
        monkeypatch.setattr(ops, "reorder_states", lambda states, slots, parents: states)
    else:
        llm.cache.reorder = lambda *a: None


def apart(outs, others):
    """For each prompt: do the two searches' hypotheses differ by other tokens, or by scores far beyond what rounding does to them?"""
    return [any(h.token_ids != k.token_ids or abs(h.score - k.score) > 1e3 * 2 * OFF * len(h.token_ids) for h, k in zip(o.hypotheses, p.hypotheses))
            for o, p in zip(outs, others)]
