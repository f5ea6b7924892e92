"""The small models that beam search is tested with: pages only, a window whose pages come back, states beside pages, states alone.  Their logits
are spread (the head's weights, or all of a tied table, times a number), so that searches have something to choose between."""
import torch

import helpers
import plain_qwen2
import plain_zazilix
import test_zazilix_gpu as zazilix


def qwen2(name):
    tensors = helpers.tiny_tensors(name, torch.float32)
    head = "lm_head.weight" if "lm_head.weight" in tensors else "model.embed_tokens.weight"
    tensors[head] = tensors[head] * 12
    cfg = helpers.tiny_config(name)
    pcfg = helpers.plain_config(cfg)
    double = {k: v.double() for k, v in tensors.items()}
    return cfg, tensors, helpers.TINY[name]["page_size"], lambda ids: plain_qwen2.forward(torch.tensor(ids), double, pcfg, torch.float64)[-1]


def recurrent(name):
    from pico_vllm_b200.registry import config_from_dict
    raw = zazilix.SHAPES[name]
    tensors = zazilix._tensors(raw, zazilix.SEEDS[name])
    tensors["head"] = tensors["head"] * 12
    return config_from_dict(raw), tensors, 8, lambda ids: plain_zazilix.forward(raw, tensors, ids)[-1]


def model(name):
    """(config, tensors, page size, next_logits in float64) of one of the small models."""
    family, which = name.split("/")
    return {"qwen2": qwen2, "recurrent": recurrent}[family](which)


# (model, prompts' lengths, beams, tokens, length penalty): prompts that end inside a page, on its border and after one token; portions; beams that
# take all slots, and one alone
SEARCHES = [("qwen2/a", (1, 16, 37), 4, 20, 1.0), ("qwen2/b", (8, 30, 5, 24), 3, 26, 0.0), ("qwen2/c", (9,), 1, 9, 1.0), ("qwen2/c", (4, 3), 8, 7, 2.0),
            ("recurrent/a", (7, 16), 3, 7, 1.0), ("recurrent/b", (10, 8, 1), 2, 8, 0.5)]


def llm(name, device, beams, at_once=2, end_token=None, dtype="float32", **options):
    config, tensors, page, _ = model(name)
    return llm_of(config, tensors, device, beams, at_once, end_token, dtype, **{"page_size": page, **options})


def llm_of(config, tensors, device, beams, at_once=2, end_token=None, dtype="float32", **options):
    from pico_vllm_b200 import LLM, EngineConfig
    from pico_vllm_b200.engine import model_from_tensors
    options = {"use_cuda_graph": False, "max_cache_tokens": 1024, "max_num_batched_tokens": 16, **options}
    ecfg = EngineConfig(dtype=dtype, device=device, max_num_seqs=at_once * beams, **options)
    m = model_from_tensors(config, tensors, ecfg)
    out = LLM(m, engine_config=ecfg)
    out.eos_token_id = out.scheduler.eos_token_id = end_token
    return out


def prompts_of(name, lengths):
    vocab = model(name)[0].vocab_size if hasattr(model(name)[0], "vocab_size") else model(name)[0].vocab
    return [helpers.random_ids(n, vocab, 300 + n) for n in lengths]
