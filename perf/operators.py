"""The operators of beam search, as cases that can be timed and compared with a plain computation.

Three of them, in the order in which one step of a search calls them: the choice of the beams that go on (log-softmax over the
vocabulary, the best of all beams together, hypotheses that end set aside), the move of the states that a request keeps in a row of
its own, and the copy of cache pages (the last, partly filled page of a beam that another one branches off from; pages that are
brought together).

``own`` says whose computation ``run`` is: the plain one below or the framework's.
"""
import math

import torch

own = False
DEV = "cuda:0"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one request of four beams over the vocabulary of the 1.5B shape: the smallest call, where latency counts
        dict(name="select_1x4", kind="select", groups=1, rows=4, beams=4, vocab=151936, end=True, pad=0, masked=0.0, dead=0),
        # sixteen prompts at their end: one row of logits each, eight beams come of it
        dict(name="select_first_16x8", kind="select", groups=16, rows=1, beams=8, vocab=152064, end=True, pad=0, masked=0.0, dead=0),
        # an odd vocabulary in rows that are wider, half of it masked, a beam of each request that holds nothing yet, and no end token
        dict(name="select_7x5_odd", kind="select", groups=7, rows=5, beams=5, vocab=49999, end=False, pad=2, masked=0.5, dead=1),
        # a full server: 64 requests of four beams
        dict(name="select_64x4", kind="select", groups=64, rows=4, beams=4, vocab=151936, end=True, pad=0, masked=0.0, dead=0),
        # one request of four beams in a model of few layers with a matrix memory and a short convolution
        dict(name="states_1x4", kind="states", entries=4, row="16x128x128", side="3x4096", dtype="float32", slots=4, groups=1, beams=4,
             moved=1, sources=1),
        # three beams with a memory whose rows hold an odd number of lines, and a single number per head beside it
        dict(name="states_5x3_odd", kind="states", entries=7, row="12x129x128", side="12", dtype="float32", slots=17, groups=5, beams=3,
             moved=2, sources=1),
        # sixteen requests of four beams in a deep model
        dict(name="states_16x4", kind="states", entries=24, row="16x128x128", side="3x4096", dtype="float32", slots=64, groups=16,
             beams=4, moved=2, sources=2),
        # the last page of one beam for three others, in all 28 layers of the 1.5B shape
        dict(name="pages_1x4", kind="pages", entries=28, tensors=2, row="2x16x128", dtype="bfloat16", pages=300, copies=3),
        # a step in which half of 256 beams branch off
        dict(name="pages_64x4", kind="pages", entries=28, tensors=2, row="2x16x128", dtype="bfloat16", pages=2100, copies=128),
        # a cache of the 7B shape brought together: a quarter of its pages moves
        dict(name="pages_together_7b", kind="pages", entries=28, tensors=2, row="4x16x128", dtype="bfloat16", pages=4000, copies=1000),
        # the 32-bit path with small pages
        dict(name="pages_float32", kind="pages", entries=12, tensors=2, row="2x8x64", dtype="float32", pages=1500, copies=333),
        # one vector per token of an odd width, pages of seven tokens: rows that start on any second byte
        dict(name="pages_latent_odd", kind="pages", entries=9, tensors=1, row="1x7x97", dtype="bfloat16", pages=5001, copies=1201),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["select", "states", "pages"])
    if kind == "select":
        beams, vocab = _log_int(rng, 2, 32), _log_int(rng, 1000, 200000)
        rows = 1 if rng.random() < 0.25 else beams
        most = 64 * 4 * 151936 // (vocab * rows)
        return dict(kind=kind, groups=_log_int(rng, 1, max(1, min(64, most))), rows=rows, beams=beams, vocab=vocab, end=rng.random() < 0.8,
                    pad=rng.choice([0, 0, 0, 1, 2, 5]), masked=rng.choice([0.0, 0.0, 0.3, 0.9]),
                    dead=rng.randint(0, rows - 1) if rng.random() < 0.2 else 0)
    if kind == "states":
        heads, vdim, dim = rng.randint(1, 16), rng.choice([16, 33, 64, 100, 128]), rng.choice([16, 48, 64, 128])
        beams, dtype = _log_int(rng, 2, 32), rng.choice(["float32", "float32", "bfloat16"])
        moved = rng.randint(1, beams - 1)
        row = heads * vdim * dim * 4
        entries = rng.randint(1, 24)
        groups = _log_int(rng, 1, max(1, min(64, 24 * 64 * (1 << 20) // (entries * row * beams))))
        return dict(kind=kind, entries=entries, row=f"{heads}x{vdim}x{dim}", side=rng.choice([f"3x{heads * 2 * dim}", f"{heads}", "3x1001"]),
                    dtype=dtype, slots=groups * beams + rng.randint(0, 5), groups=groups, beams=beams, moved=moved,
                    sources=rng.randint(1, min(moved, beams - moved)))
    entries, tensors, dtype = rng.randint(1, 36), rng.choice([1, 2, 2]), rng.choice(["bfloat16", "bfloat16", "float32"])
    heads, page, width = rng.choice([1, 2, 4, 8]), rng.choice([1, 7, 8, 16, 16, 32]), rng.choice([64, 97, 128, 128, 320, 576])
    row = entries * tensors * heads * page * width * (4 if dtype == "float32" else 2)
    copies = _log_int(rng, 1, max(1, min(3000, 900_000_000 // row)))
    return dict(kind=kind, entries=entries, tensors=tensors, row=f"{heads}x{page}x{width}", dtype=dtype,
                pages=2 * copies + rng.randint(0, min(1000, 1 + 900_000_000 // row)), copies=copies)


def _shape(text):
    return tuple(int(n) for n in text.split("x"))


# ---------------------------------------------------------------------------------------------------------- the inputs
def _rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _select_inputs(c, seed):
    """Logits as a language model's: a broad bell with a few dozen likely tokens in each row, the end token among them in every third row;
    scores of beams some tokens long.  Masked tokens and beams that hold nothing have the value minus infinity."""
    g = _rng(seed)
    R, V = c["groups"] * c["rows"], c["vocab"]
    wide = torch.randn((R, V + c["pad"]), generator=g, device=DEV).mul_(2.0)
    x = wide[:, :V]
    likely = torch.randint(0, V, (R, 40), generator=g, device=DEV)
    x.scatter_reduce_(1, likely, 6.0 + 6.0 * torch.rand((R, 40), generator=g, device=DEV), "amax")
    end = V // 2 if c["end"] else -1
    if c["masked"]:
        x.masked_fill_(torch.rand((R, V), generator=g, device=DEV) < c["masked"], -math.inf)
    if c["end"]:
        x[:, end] = torch.where(torch.rand(R, generator=g, device=DEV) < 0.34, 12.5, 0.0)
    scores = -20.0 - 4.0 * torch.rand((c["groups"], c["rows"]), generator=g, device=DEV)
    if c["dead"]:
        scores[:, c["rows"] - c["dead"]:] = -math.inf
    return x, scores, end


def _family(c, seed):
    """Slots of the groups' beams in any order, and parents: of each group's places ``moved`` take over the state of another one, of ``sources``
    different ones in all."""
    g = torch.Generator().manual_seed(seed)
    slots = torch.randperm(c["slots"], generator=g)[:c["groups"] * c["beams"]].view(c["groups"], c["beams"])
    order = torch.rand((c["groups"], c["beams"]), generator=g).argsort(1)
    taken, origin = order[:, :c["moved"]], order[:, c["moved"]:c["moved"] + c["sources"]]
    parents = torch.arange(c["beams"]).repeat(c["groups"], 1)
    parents.scatter_(1, taken, origin[:, torch.arange(c["moved"]) % c["sources"]])
    return slots.to(torch.int32).to(DEV), parents.to(torch.int32).to(DEV)


def _state_inputs(c, seed):
    g = _rng(seed)
    return [torch.randn((c["entries"], c["slots"]) + _shape(s), generator=g, device=DEV, dtype=DTYPES[t])
            for s, t in ((c["row"], c["dtype"]), (c["side"], "float32"))]


def _page_inputs(c, seed):
    g = _rng(seed)
    caches = [torch.randn((c["entries"], c["pages"]) + _shape(c["row"]), generator=g, device=DEV, dtype=DTYPES[c["dtype"]])
              for _ in range(c["tensors"])]
    order = torch.randperm(c["pages"], generator=torch.Generator().manual_seed(seed))[:2 * c["copies"]].to(torch.int32).to(DEV)
    return caches, order[:c["copies"]].contiguous(), order[c["copies"]:].contiguous()


def prepare(case, seed):
    if case["kind"] == "select":
        return case, _select_inputs(case, seed)
    if case["kind"] == "states":
        return case, (_state_inputs(case, seed),) + _family(case, seed)
    return case, _page_inputs(case, seed)


# ---------------------------------------------------------------------------------------------------------- one pass
def run(state):
    c, given = state
    if own:
        from pico_vllm_b200 import ops
        if c["kind"] == "select":
            logits, scores, end = given
            return ops.beam_select(logits, scores, c["beams"], None if end < 0 else end)
        if c["kind"] == "states":
            ops.reorder_states(*given)
        else:
            ops.copy_pages(*given)
        return given[0]
    if c["kind"] == "select":
        return _plain_select(*given, c["beams"])
    return _plain_states(*given) if c["kind"] == "states" else _plain_pages(*given)


def _plain_select(x, scores, end, beams):
    G, rows = scores.shape
    R, V = x.shape
    K = beams if end < 0 else 2 * beams
    # the normaliser: exponentials in 32 bits, their sum in 64 (beams are compared with one another by it)
    top = x.amax(1, keepdim=True)
    lse = top[:, 0].double() + torch.exp(x - top).sum(1, dtype=torch.float64).log()
    # the K best of a row, of equal ones the first: whole numbers that are ordered as (logit, -index)
    bits = (x + 0.0).view(torch.int32)
    key = (torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32) | (V - 1 - torch.arange(V, device=x.device))
    key = torch.topk(key, min(K, V), dim=1).values
    token = V - 1 - (key & 0xffffffff)
    value = x.gather(1, token).double() + (scores.reshape(R).double() - lse)[:, None]
    # the K best of a group: by value, of equal ones the first of all its rows' tokens
    flat = (token + V * (torch.arange(R, device=x.device) % rows)[:, None]).view(G, -1)
    value = torch.where(value.isfinite(), value, -math.inf).view(G, -1)
    flat, at = flat.sort(1)
    value, at = value.gather(1, at).sort(dim=1, descending=True, stable=True)
    pad = max(0, K - value.shape[1])
    value = torch.nn.functional.pad(value[:, :K], (0, pad), value=-math.inf)
    flat = torch.nn.functional.pad(flat.gather(1, at)[:, :K], (0, pad))
    alive = value > -math.inf
    token, parent = flat % V, flat // V
    # hypotheses that end, among the best ones
    place = torch.arange(beams, device=x.device)
    ends = (alive & (token == end))[:, :beams, None] & (parent[:, :beams, None] == torch.arange(rows, device=x.device))
    ended = torch.where(ends, value[:, :beams, None], -math.inf).amax(1)
    # those that go on, best first
    going = alive & (token != end)
    pick = (~(going & (going.cumsum(1) <= beams))).to(torch.int32).sort(dim=1, stable=True).indices[:, :beams]
    token, parent, value, alive = (t.gather(1, pick) for t in (token, parent, value, going))
    # the first child of a parent stays at its place, the others take the places that are left
    same = (parent[:, :, None] == parent[:, None, :]) & alive[:, None, :]
    first = alive & ~same.tril(-1).any(2)
    left = ((parent[:, :, None] == place) & first[:, :, None]).any(1).to(torch.int32).sort(dim=1, stable=True).indices
    at = torch.where(first, parent, left.gather(1, ((~first).cumsum(1) - 1).clamp(min=0)))
    token, parent = torch.where(alive, token, -1), torch.where(alive, parent, at)
    back = at.sort(1).indices
    return (token.gather(1, back).to(torch.int32), parent.gather(1, back).to(torch.int32),
            torch.where(alive, value, -math.inf).gather(1, back).float(), ended.float())


def _plain_states(states, slots, parents):
    at, source = slots.long().view(-1), slots.long().gather(1, parents.long()).view(-1)
    at, source = at[at != source], source[at != source]
    return [t.index_copy_(1, at, t.index_select(1, source)) for t in states]


def _plain_pages(caches, src, dst):
    src, dst = src.long(), dst.long()
    return [t.index_copy_(1, dst, t.index_select(1, src)) for t in caches]


# ---------------------------------------------------------------------------------------------------------- what it takes
def work(case):
    c = case
    if c["kind"] == "select":
        n = c["groups"] * c["rows"]
        # a logit is subtracted from, raised, added and compared
        return {"bytes": 4 * (n * c["vocab"] + n + c["groups"] * (3 * c["beams"] + c["rows"])), "flops": 4 * n * c["vocab"]}
    size = 4 if c["dtype"] == "float32" else 2
    if c["kind"] == "states":
        row = c["entries"] * (math.prod(_shape(c["row"])) * size + math.prod(_shape(c["side"])) * 4)
        return {"bytes": c["groups"] * ((c["moved"] + c["sources"]) * row + 8 * c["beams"]), "flops": 0}
    return {"bytes": c["copies"] * (2 * c["entries"] * c["tensors"] * math.prod(_shape(c["row"])) * size + 8), "flops": 0}


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    c = case
    if c["kind"] == "pages":
        caches, src, dst = _page_inputs(c, seed)
        for t in caches:
            for s, d in zip(src.tolist(), dst.tolist()):
                t[:, d].copy_(t[:, s])
        return caches
    if c["kind"] == "states":
        states, (slots, parents) = _state_inputs(c, seed), (t.tolist() for t in _family(c, seed))
        for t in states:
            before = t.clone()
            for line, family in zip(slots, parents):
                for slot, parent in zip(line, family):
                    t[:, slot] = before[:, line[parent]]
        return states
    x, scores, end = _select_inputs(c, seed)
    B, rows, V = c["beams"], c["rows"], c["vocab"]
    tokens, parents, news, endeds = [], [], [], []
    for g in range(c["groups"]):
        logp = x[g * rows:(g + 1) * rows].double().log_softmax(1) + scores[g].double()[:, None]
        value, flat = logp.flatten().sort(descending=True, stable=True)
        value, flat = value[:2 * B].tolist(), flat[:2 * B].tolist()
        ranked = [(v, f // V, f % V) for v, f in zip(value, flat) if math.isfinite(v)][:2 * B if end >= 0 else B]
        ended = [-math.inf] * rows
        for v, parent, token in ranked[:B]:
            if token == end:
                ended[parent] = v
        places, spare = [None] * B, []
        for v, parent, token in [r for r in ranked if r[2] != end][:B]:
            if places[parent] is None:
                places[parent] = (v, parent, token)
            else:
                spare.append((v, parent, token))
        for p in range(B):
            if places[p] is None:
                places[p] = spare.pop(0) if spare else (-math.inf, p, -1)
        tokens.append([p[2] for p in places])
        parents.append([p[1] for p in places])
        news.append([p[0] for p in places])
        endeds.append(ended)
    i32, f64 = dict(dtype=torch.int32, device=DEV), dict(dtype=torch.float64, device=DEV)
    return torch.tensor(tokens, **i32), torch.tensor(parents, **i32), torch.tensor(news, **f64), torch.tensor(endeds, **f64)
