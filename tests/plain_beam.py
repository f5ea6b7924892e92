"""Beam search's operators restated plainly: the choice of beams in float64, rows moved one by one."""
import math

import torch


def candidates(logits, scores, most):
    """[(value, beam, token), ..] of one request, the best ``most``, best first: logits [rows, V], scores [rows], in float64."""
    rows, V = logits.shape
    x = logits.double()
    top = x.amax(1, keepdim=True)
    # equal rows are to have equal sums: all start alike, on a multiple of 512 numbers, so that they are added up in one order
    terms = torch.nn.functional.pad((x - top).exp(), (0, -V % 512))
    lp = ((x - top) - terms.sum(1, keepdim=True).log()) + scores.double()[:, None]
    lp = lp.flatten().nan_to_num(-math.inf, -math.inf, -math.inf)
    value, flat = lp.sort(descending=True, stable=True)
    return [(v, f // V, f % V) for v, f in zip(value[:most].tolist(), flat[:most].tolist()) if math.isfinite(v)]


def select(logits, scores, beams, end_token=None):
    """(tokens, parents, scores, ended) lists of one request, and the ranked candidates that decided them with the next one."""
    rows = logits.shape[0]
    most = beams if end_token is None else 2 * beams
    further = candidates(logits, scores, most + 1)
    ranked = further[:most]
    ended = [-math.inf] * rows
    for v, b, t in ranked[:beams]:
        if t == end_token:
            ended[b] = v
    places, spare = [None] * beams, []
    for c in [c for c in ranked if c[2] != end_token][:beams]:
        if places[c[1]] is None:
            places[c[1]] = c
        else:
            spare.append(c)
    for p in range(beams):
        if places[p] is None:
            places[p] = spare.pop(0) if spare else (-math.inf, p, -1)
    return [c[2] for c in places], [c[1] for c in places], [c[0] for c in places], ended, further


def reorder(t, slots, parents):
    """t [entries, slots, ...] after t[:, slots[g][p]] = old t[:, slots[g][parents[g][p]]]."""
    new = t.clone()
    for line, family in zip(slots, parents):
        for slot, parent in zip(line, family):
            new[:, slot] = t[:, line[parent]]
    return new


def copy(t, src, dst):
    new = t.clone()
    for s, d in zip(src, dst):
        if s >= 0 and d >= 0:
            new[:, d] = t[:, s]
    return new
