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


def search(next_logits, prompt, beams, max_new, end_token=None, length_penalty=1.0):
    """Beam search over ``next_logits(tokens) -> [V]``: [(value, score, tokens, reason), ..] best first, and the smallest distance of two
    values that were compared (inputs on which rounding decides are none to test with)."""
    found, near = [], math.inf
    paths, scores = [[]], [0.0]

    def keep(tokens, score, reason):
        value = score / len(tokens) ** length_penalty
        if len(found) >= beams and value <= found[-1][0]:
            return
        found.append((value, score, tokens, reason))
        found.sort(key=lambda h: -h[0])
        del found[beams:]
    for n in range(1, max_new + 1):
        logits = torch.stack([next_logits(prompt + p) if p is not None else torch.zeros_like(next_logits(prompt)) for p in paths])
        tokens, parents, new, ended, ranked = select(logits.double(), torch.tensor(scores, dtype=torch.float64), beams, end_token)
        near = min([near] + [a[0] - b[0] for a, b in zip(ranked, ranked[1:])])
        for p, v in zip(paths, ended):
            if v > -math.inf:
                keep(p + [end_token], v, "eos")
        paths = [paths[q] + [t] if t >= 0 else None for t, q in zip(tokens, parents)]
        scores = new
        if n == max_new:
            for p, v in zip(paths, scores):
                if v > -math.inf:
                    keep(p, v, "length")
            break
        if max(scores) == -math.inf:
            break
        if len(found) >= beams:
            gap = max(scores) / n ** length_penalty - found[-1][0]
            near = min(near, abs(gap))
            if gap <= 0:
                break
    return found, near
