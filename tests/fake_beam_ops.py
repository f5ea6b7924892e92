"""Test doubles of the kernels of beam search, beside those of fake_ops.py."""
import torch

import plain_beam as plain


def beam_select(logits, scores, beams, end_token=None, out=None):
    G, rows = scores.shape
    out = torch.empty(G * (3 * beams + rows), dtype=torch.int32) if out is None else out
    c, floats = G * beams, out.view(torch.float32)
    found = out[:c].view(G, beams), out[c:2 * c].view(G, beams), floats[2 * c:3 * c].view(G, beams), floats[3 * c:].view(G, rows)
    for g in range(G):
        got = plain.select(logits[g * rows:(g + 1) * rows], scores[g].clone(), beams, end_token)
        for t, v in zip(found, got):
            t[g] = torch.tensor(v, dtype=t.dtype)
    return found


def copy_pages(tensors, src, dst):
    for t in tensors:
        t.copy_(plain.copy(t, src.tolist(), dst.tolist()))
    return tensors


def reorder_states(states, slots, parents):
    for t in states:
        t.copy_(plain.reorder(t, slots.tolist(), parents.tolist()))
    return states


def install(monkeypatch):
    import pico_vllm_b200.ops as ops
    for name in ("beam_select", "copy_pages", "reorder_states"):
        monkeypatch.setattr(ops, name, globals()[name])
