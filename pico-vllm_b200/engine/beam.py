"""Beam search over the step function.

A search holds one cache slot per beam.  Its prompt runs once, in one slot; then the slot branches (``CacheManager.fork``: full pages
are shared, the last one and the states copied), and from there every step is one token of every beam of every search, one choice
(``ops.beam_select``) and one ``CacheManager.reorder``.  The choice leaves the best child of a beam in the beam's place, so that what moves is
only what beams that die make room for.  The host reads the chosen tokens before the next step: block tables are made there.

The reference has no beam search.
"""
from __future__ import annotations

import math
from collections import deque
from dataclasses import dataclass, field
from typing import Deque, List, Optional, Sequence, Tuple

import torch

from .. import ops
from ..errors import ConfigError, ScheduleError
from ..sampling import BeamParams
from .runner import StepItem


@dataclass
class Hypothesis:
    token_ids: List[int]             # the generated tokens, the end token included
    score: float                     # sum of their log-probabilities
    value: float                     # what it is ranked by: score / length ** length_penalty
    finish_reason: str               # "eos" or "length"
    text: Optional[str] = None       # generated text, when the folder has a tokenizer


@dataclass
class BeamOutput:
    prompt_token_ids: List[int]
    hypotheses: List[Hypothesis]     # best first


@dataclass
class _Search:
    prompt: List[int]
    reserved: List[int]                                        # pages of each group that it may come to hold
    slots: List[int] = field(default_factory=list)
    computed: int = 0                                          # prompt tokens in the cache
    length: int = 0                                            # tokens generated
    paths: List[Optional[tuple]] = field(default_factory=list)  # per place: (path before, token)
    scores: List[float] = field(default_factory=list)
    found: List[Hypothesis] = field(default_factory=list)      # those that have ended, best first, no more than beams


def _path_tokens(path: Optional[tuple]) -> List[int]:
    out: List[int] = []
    while path is not None:
        path, token = path
        out.append(token)
    return out[::-1]


class BeamSearch:
    """Runs prompts to the end with one set of parameters.  The engine has to be idle: slots and pages are taken by what they may
    come to, which requests of another kind know nothing of."""

    def __init__(self, runner, cache, cfg, params: BeamParams, end_token: Optional[int]):
        self.runner, self.cache, self.cfg, self.params = runner, cache, cfg, params
        vocab = runner.model.vocab_size
        self.end = end_token if not params.ignore_eos and end_token is not None and 0 <= end_token < vocab else None
        self.steps = self.prefill_tokens = self.decode_tokens = 0
        B = params.beams
        if B > cache.max_num_seqs or B > cfg.max_num_batched_tokens:
            raise ConfigError(f"{B} beams need as many slots and as large a token budget (max_num_seqs {cache.max_num_seqs}, "
                              f"max_num_batched_tokens {cfg.max_num_batched_tokens})")
        self._host = None
        self._held: Tuple[tuple, Optional[torch.Tensor], Optional[torch.Tensor]] = ((), None, None)

    # ------------------------------------------------------------------ all of it
    def run(self, prompts: Sequence[List[int]]) -> List[List[Hypothesis]]:
        searches = [_Search(p, self._pages(len(p))) for p in prompts]
        waiting: Deque[_Search] = deque(searches)
        active: List[_Search] = []
        try:
            while waiting or active:
                self._admit(waiting, active)
                self._prompts([s for s in active if not s.scores])
                going = [s for s in active if s.scores]
                if going:
                    self._tokens(going)
                for s in [s for s in active if s.scores and self._over(s)]:
                    self._free(s)
                    active.remove(s)
        finally:
            for s in active:
                self._free(s)
        ops.check_kernel_status()
        return [s.found[:self.params.num_return] for s in searches]

    def _pages(self, n: int) -> List[int]:
        """Pages of each group that a search over a prompt of n tokens may come to hold: the prompt's full ones once, what follows for every beam.
        (The last token is never computed.)"""
        ps, B = self.cache.page_size, self.params.beams
        last = -(-(n + self.params.max_new_tokens - 1) // ps)
        return [last + (B - 1) * (last - n // ps) for _ in self.cache.groups]

    def _admit(self, waiting, active) -> None:
        B = self.params.beams
        while waiting and (len(active) + 1) * B <= min(self.cache.max_num_seqs, self.cfg.max_num_batched_tokens):
            s = waiting[0]
            fits = all(need + sum(a.reserved[i] for a in active) <= g.pool.num_pages
                       for i, (need, g) in enumerate(zip(s.reserved, self.cache.groups)))
            if active and not fits:
                return                  # (alone it may try: beams that go the same way share more than the bound says)
            s.slots = [self.cache.acquire(s)]
            active.append(waiting.popleft())

    def _free(self, s: _Search) -> None:
        for slot in s.slots:
            self.cache.release(slot)
        s.slots = []

    # ------------------------------------------------------------------ prompts, in portions
    def _prompts(self, todo: List[_Search]) -> None:
        budget = self.cfg.max_num_batched_tokens
        chunk = self.cfg.prefill_chunk or budget
        items, ended = [], []
        for s in todo:
            n = min(len(s.prompt) - s.computed, chunk, budget)
            if n <= 0:
                break
            last = s.computed + n == len(s.prompt)
            items.append(StepItem(s.slots[0], s.prompt[s.computed:s.computed + n], (n - 1,) if last else ()))
            s.computed += n
            budget -= n
            self.prefill_tokens += n
            if last:
                ended.append(s)
        if not items:
            return
        logits = self.runner.step(items)
        self.steps += 1
        if not ended:
            return
        for s in ended:
            s.scores, s.paths = [0.0], [None]
        self._choose(ended, logits, torch.zeros((len(ended), 1), dtype=torch.float32, device=logits.device))
        for s in ended:
            if not self._over(s):       # (what is over needs no branches)
                s.slots += self.cache.fork(s.slots[0], self.params.beams - 1, [s] * (self.params.beams - 1))

    # ------------------------------------------------------------------ one token of every beam
    def _tokens(self, going: List[_Search]) -> None:
        going = [s for s in going if not self._over(s)]
        if not going:
            return
        # (a place that holds nothing goes along with any token)
        items = [StepItem(slot, (path[1] if path is not None else 0,), (0,)) for s in going for slot, path in zip(s.slots, s.paths)]
        logits = self.runner.step(items)
        self.steps += 1
        self.decode_tokens += len(items)
        key = tuple(id(s) for s in going)
        if self._held[0] != key:
            host = torch.tensor([s.scores for s in going], dtype=torch.float32)
            slots = torch.tensor([s.slots for s in going], dtype=torch.int32)
            self._held = (key, slots.to(self.cache.device, non_blocking=True), host.to(self.cache.device, non_blocking=True))
        _, slots, scores = self._held
        families, parents, scores = self._choose(going, logits, scores)
        self._held = (key, slots, scores)
        alive = [i for i, s in enumerate(going) if not self._over(s)]
        if len(alive) == len(going):
            self.cache.reorder([s.slots for s in going], families, (slots, parents))
        else:
            self.cache.reorder([going[i].slots for i in alive], [families[i] for i in alive])

    def _choose(self, searches: List[_Search], logits: torch.Tensor, scores: torch.Tensor):
        """The next tokens, places and scores of the searches, and the hypotheses that end.  Returns the parents (here and on the device) and
        the scores on the device."""
        B, rows = self.params.beams, scores.shape[1]
        n = len(searches)
        out = torch.empty(n * (3 * B + rows), dtype=torch.int32, device=logits.device)
        tokens, parents, new, _ = ops.beam_select(logits, scores, B, self.end, out)
        if self._host is None or self._host.numel() < out.numel():
            self._host = torch.empty(max(256, out.numel()), dtype=torch.int32, pin_memory=out.is_cuda)
        host = self._host[:out.numel()]
        host.copy_(out, non_blocking=True)
        if out.is_cuda:
            torch.cuda.current_stream().synchronize()
        c = n * B
        toks, fams = host[:c].view(n, B).tolist(), host[c:2 * c].view(n, B).tolist()
        floats = host.view(torch.float32)
        values, ended = floats[2 * c:3 * c].view(n, B).tolist(), floats[3 * c:].view(n, rows).tolist()
        for s, tok, family, value, ends in zip(searches, toks, fams, values, ended):
            s.length += 1
            for path, v in zip(s.paths, ends):
                if v > -math.inf:
                    self._end(s, (path, self.end), v, "eos")
            s.paths = [(s.paths[q], t) if t >= 0 else None for t, q in zip(tok, family)]
            s.scores = value
            if s.length >= self.params.max_new_tokens:
                for path, v in zip(s.paths, value):
                    if v > -math.inf:
                        self._end(s, path, v, "length")
        return fams, parents, new

    def _value(self, score: float, length: int) -> float:
        return score / length ** self.params.length_penalty

    def _end(self, s: _Search, path: tuple, score: float, reason: str) -> None:
        value = self._value(score, s.length)
        if len(s.found) >= self.params.beams and value <= s.found[-1].value:
            return
        s.found.append(Hypothesis(_path_tokens(path), score, value, reason))
        s.found.sort(key=lambda h: -h.value)       # (stable: of equal ones the earlier first)
        del s.found[self.params.beams:]

    def _over(self, s: _Search) -> bool:
        """All tokens generated, no beam left, or as many ended hypotheses as beams and no beam that is worth more now than the worst of them."""
        best = max(s.scores)
        if s.length >= self.params.max_new_tokens or best == -math.inf:
            return True
        return s.length > 0 and len(s.found) >= self.params.beams and self._value(best, s.length) <= s.found[-1].value


def beam_search(llm, prompts, params: BeamParams) -> List[BeamOutput]:
    """``LLM.beam_search``."""
    if llm.scheduler.has_work() or llm._pending is not None:
        raise ScheduleError("beam search needs the engine to itself: finish the requests that were submitted first")
    ids = [llm._encode(p) for p in prompts]
    for p in ids:
        if not p:
            raise ScheduleError("a request needs at least one prompt token")
        if len(p) + params.max_new_tokens > llm.cache.max_seq_len:
            raise ScheduleError(f"prompt ({len(p)}) + max_new_tokens ({params.max_new_tokens}) exceeds the longest request the cache "
                                f"holds ({llm.cache.max_seq_len})")
    search = BeamSearch(llm.runner, llm.cache, llm.cfg, params, llm.eos_token_id)
    found = search.run(ids)
    llm.stats["steps"] += search.steps
    llm.stats["prefill_tokens"] += search.prefill_tokens
    llm.stats["decode_tokens"] += search.decode_tokens
    if llm.tokenizer is not None:
        for hyps in found:
            for h in hyps:
                h.text = llm._decode(h.token_ids)
    return [BeamOutput(p, h) for p, h in zip(ids, found)]
