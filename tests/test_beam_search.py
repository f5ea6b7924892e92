"""Beam search, and the cache's branches, on the CPU with the kernels replaced by torch doubles: the choice, the order of steps, block tables, shared
pages, states passed on, what is refused."""
import random

import pytest
import torch

import beam_models
import fake_beam_ops
import fake_ops
import plain_beam
from pico_vllm_b200.cache import CacheManager, PagePool
from pico_vllm_b200.errors import ConfigError, OutOfPages, PicoError, ScheduleError
from pico_vllm_b200.parts import FixedState, PagedKV


@pytest.fixture
def on_cpu(monkeypatch):
    fake_ops.install(monkeypatch)
    fake_beam_ops.install(monkeypatch)
    import pico_vllm_b200.engine.core as core
    monkeypatch.setattr(core, "_require_device", lambda device: None)


def compare(outs, prompts, next_logits, beams, tokens, end, penalty, off):
    """The hypotheses are the plain search's, in its order; scores as near as logits that are off by ``off`` make them (two of them a token: the token's own and
    the normaliser)."""
    for p, o in zip(prompts, outs):
        want, near = plain_beam.search(next_logits, p, beams, tokens, end, penalty)
        assert near > 5e-5, f"inputs too near a tie: {near}"         # (32-bit logits are off by some 1e-6 here)
        assert [h.token_ids for h in o.hypotheses] == [w[2] for w in want]
        assert [h.finish_reason for h in o.hypotheses] == [w[3] for w in want]
        for h, w in zip(o.hypotheses, want):
            assert abs(h.score - w[1]) <= 2 * off * len(w[2]) + abs(w[1]) * 2.0 ** -23
            assert abs(h.value - h.score / len(h.token_ids) ** penalty) <= 1e-9 * abs(h.value)
        assert o.prompt_token_ids == p


@pytest.mark.parametrize("name,lengths,beams,tokens,penalty", beam_models.SEARCHES)
@pytest.mark.parametrize("ends", [False, True])
def test_search_equals_plain(on_cpu, name, lengths, beams, tokens, penalty, ends):
    from pico_vllm_b200 import BeamParams
    prompts = beam_models.prompts_of(name, lengths)
    next_logits = beam_models.model(name)[3]
    end = None
    if ends:                # a token that some hypotheses come to
        end = plain_beam.search(next_logits, prompts[0], beams, tokens, None, penalty)[0][0][2][min(3, tokens - 1)]
    llm = beam_models.llm(name, "cpu", beams, end_token=end)
    outs = llm.beam_search(prompts, BeamParams(beams=beams, max_new_tokens=tokens, length_penalty=penalty))
    compare(outs, prompts, next_logits, beams, tokens, end, penalty, 2e-5)
    llm.cache.check()
    assert all(g.pool.in_use == 0 for g in llm.cache.groups) and llm.cache.free_slots == llm.cache.max_num_seqs


# ------------------------------------------------------------------ the cache's branches
FULL, WIN = PagedKV(1, 2, None), PagedKV(2, 2, 9)
STATES = (FixedState((3, 2)), FixedState((5,)), FixedState((3, 2)), FixedState((0, 4)))


def _manager(num_pages=60, slots=8, page=4, entries=(FULL, WIN, FULL) + STATES, allocate=True):
    return CacheManager(list(entries), page, num_pages, slots, 80, torch.float32, "cpu", allocate=allocate, poison_freed=True)


class _Told:
    """What every slot should hold, written token by token."""

    def __init__(self, m):
        self.m, self.text, self.next = m, {}, 1.0

    def write(self, slot, n):
        m = self.m
        start = m.append(slot, n)
        marks = []
        for i in range(n):
            marks.append(self.next)
            self.next += 1.0
        for gi, g in enumerate(m.groups):
            for pos, row, mark in zip(range(start, start + n), m.slot_mapping(gi, slot, start, n), marks):
                for t in g.tensors.values():
                    t[:, row // m.page_size, :, row % m.page_size] = mark
        for s in m.states.values():
            s[slot] = marks[-1]
        m.commit(slot)
        self.text[slot] = self.text.get(slot, []) + marks

    def check(self):
        m = self.m
        m.check()
        for slot, marks in self.text.items():
            assert m.seq_len[slot] == len(marks)
            for gi, g in enumerate(m.groups):
                first = 0 if g.spec.window is None else max(0, len(marks) + 1 - g.spec.window)
                for pos in range(first, len(marks)):
                    row = m.slot_mapping(gi, slot, pos, 1)[0]
                    for t in g.tensors.values():
                        assert (t[:, row // m.page_size, :, row % m.page_size] == marks[pos]).all()
            for s in m.states.values():
                assert (s[slot] == marks[-1]).all()


@pytest.mark.parametrize("seed", range(6))
def test_branches_hold_what_they_should_in_any_order(on_cpu, seed):
    """Families that branch, are reordered in any way (children of one, cycles), grow, end and are brought together: every slot holds its own
    text, full pages are shared, no page is lost."""
    rng = random.Random(seed)
    m = _manager()
    told, families = _Told(m), []
    for _ in range(60):
        op = rng.choice(["new", "grow", "grow", "grow", "reorder", "reorder", "end", "compact"])
        if op == "new" and m.free_slots >= 3:
            n = rng.randint(1, min(4, m.free_slots))
            slot = m.acquire("r")
            told.write(slot, rng.randint(1, 14))
            forks = m.fork(slot, n - 1)
            for s in forks:
                told.text[s] = list(told.text[slot])
            families.append([slot] + forks)
            L = len(told.text[slot])
            for g in m.groups:          # full pages are shared
                first = int(g.first_block[slot])
                assert all((g.tables[s, first:L // 4] == g.tables[slot, first:L // 4]).all() for s in forks)
        elif op == "grow" and families:
            for slot in rng.choice(families):
                if len(told.text[slot]) < 60:
                    told.write(slot, 1)
        elif op == "reorder" and families:
            some = rng.sample(families, rng.randint(1, len(families)))
            parents = [[rng.randrange(len(f)) for _ in f] for f in some]
            held = [g.pool.available for g in m.groups]
            texts = {s: told.text[f[q]] for f, p in zip(some, parents) for s, q in zip(f, p)}
            m.reorder(some, parents)
            told.text.update({s: list(t) for s, t in texts.items()})
            assert all(g.pool.available >= n for g, n in zip(m.groups, held))       # needs no page
        elif op == "end" and len(families) > 1:
            for slot in families.pop(rng.randrange(len(families))):
                m.release(slot)
                del told.text[slot]
        elif op == "compact":
            m.compact()
            assert all(sorted(g.pool._free) == list(range(g.pool.in_use, g.pool.num_pages)) for g in m.groups)
        told.check()
    for f in families:
        for slot in f:
            m.release(slot)
    m.check()
    assert all(g.pool.in_use == 0 for g in m.groups)


def test_states_of_equal_entries_lie_together():
    m = _manager()
    assert [tuple(t.shape) for t in m.state_stacks] == [(2, 8, 3, 2), (1, 8, 5), (1, 8, 0, 4)]
    assert m.states[3].data_ptr() == m.state_stacks[0][0].data_ptr() and m.states[5].data_ptr() == m.state_stacks[0][1].data_ptr()
    assert all(s.is_contiguous() and s.shape[0] == 8 for s in m.states.values())
    assert m.states[5].data_ptr() % 512 == m.states[3].data_ptr() % 512


def test_branches_refused_and_nothing_taken():
    m = _manager(num_pages=8, entries=(FULL,), allocate=False)
    a = m.acquire("a")
    m.append(a, 10)
    with pytest.raises(PicoError, match="not committed"):
        m.fork(a, 1)
    with pytest.raises(PicoError, match="not committed"):
        m.compact()
    m.commit(a)
    with pytest.raises(PicoError, match="not held"):
        m.fork(a + 1 if a + 1 < 8 else a - 1, 1)
    with pytest.raises(PicoError, match="owner"):
        m.fork(a, 2, ["one"])
    with pytest.raises(PicoError):
        m.fork(a, -1)
    with pytest.raises(ScheduleError):
        m.fork(a, 8)
    with pytest.raises(OutOfPages):
        m.fork(a, 6)                # 3 of 8 pages held, a copy of the last one each
    assert m.fork(a, 0) == [] and m.groups[0].pool.in_use == 3 and m.free_slots == 7
    b, c = m.fork(a, 2)
    assert m.groups[0].pool.in_use == 5 and m.owner[b] is True
    m.append(b, 1)
    for slots, parents, match in (([[a, b, c]], [[0, 1, 1]], "committed"), ([[a, c], [c]], [[0, 1], [0]], "one family"), ([[a, c]], [[0]], "parent in it"),
                                  ([[a, c]], [[0, 2]], "parent in it"), ([[a, c]], [], "has its parents")):
        with pytest.raises(PicoError, match=match):
            m.reorder(slots, parents)
    m.commit(b)
    with pytest.raises(PicoError, match="equally many"):
        m.reorder([[a, b]], [[1, 0]])
    m.check()


def test_pages_moved_or_refused():
    pool = PagePool(6)
    pool.allocate(6)
    pool.share([5])
    pool.release([0, 2, 3])
    assert pool.gather_plan() == ([4, 5], [0, 2])
    for src, dst in (([4], [1]), ([3], [0]), ([4, 5], [0]), ([4, 4], [0, 2]), ([4, 5], [0, 0]), ([6], [0])):
        with pytest.raises(PicoError):
            pool.move(src, dst)
    pool.move([4, 5], [0, 2])
    assert [pool.refcount(p) for p in range(6)] == [1, 1, 2, 0, 0, 0] and pool.allocate(3) == [3, 4, 5]


# ------------------------------------------------------------------ the entry point
def test_requests_and_searches_one_after_the_other(on_cpu):
    """The engine generates as before beside searches, whose pages and slots come back; pages brought together between steps change no token."""
    from pico_vllm_b200 import BeamParams, SamplingParams
    prompts = beam_models.prompts_of("qwen2/a", (5, 21))
    llm = beam_models.llm("qwen2/a", "cpu", 3)
    sp = SamplingParams(temperature=0.0, max_new_tokens=9, ignore_eos=True)
    want = [o.token_ids for o in llm.generate(prompts, sp)]
    hyps = llm.beam_search(prompts, BeamParams(beams=3, max_new_tokens=5))
    assert [o.token_ids for o in llm.generate(prompts, sp)] == want
    assert llm.beam_search(prompts, BeamParams(beams=3, max_new_tokens=5)) == hyps
    one = llm.beam_search(prompts[0], BeamParams(beams=1, max_new_tokens=9, ignore_eos=True))
    assert one[0].hypotheses[0].token_ids == want[0]             # one beam is greedy
    few = llm.beam_search(prompts, BeamParams(beams=3, max_new_tokens=5, num_return=2))
    assert [o.hypotheses for o in few] == [o.hypotheses[:2] for o in hyps]
    assert llm.beam_search([], BeamParams(beams=3)) == []
    # a short request ends while a long one goes on; its pages lie below
    short = llm.submit(prompts[1], max_new_tokens=2, temperature=0.0, ignore_eos=True)
    long = llm.submit(prompts[0], max_new_tokens=9, temperature=0.0, ignore_eos=True)
    with pytest.raises(ScheduleError, match="itself"):
        llm.beam_search(prompts, BeamParams(beams=3))
    llm.mark_finished()
    done, copied = {}, 0
    while not llm.is_done():
        done.update(llm.step())
        copied += llm.compact_cache()
        llm.cache.check()
    assert done[long] == prompts[0] + want[0] and done[short] == prompts[1] + want[1][:2] and copied > 0


@pytest.mark.parametrize("end_at", [None, 0, 2])
def test_a_single_token(on_cpu, end_at):
    """Nothing branches: the choice after the prompt is all, the end token among it or not."""
    from pico_vllm_b200 import BeamParams
    prompts = beam_models.prompts_of("qwen2/a", (16, 5))
    next_logits = beam_models.model("qwen2/a")[3]
    lp = next_logits(prompts[0]).log_softmax(0).sort(descending=True)
    end = None if end_at is None else int(lp.indices[end_at])
    llm = beam_models.llm("qwen2/a", "cpu", 4, end_token=end)
    outs = llm.beam_search(prompts, BeamParams(beams=4, max_new_tokens=1))
    compare(outs, prompts, next_logits, 4, 1, end, 1.0, 2e-5)
    if end is not None:
        assert [h.finish_reason for h in outs[0].hypotheses] == ["eos" if k == end_at else "length" for k in range(4)]
    llm.cache.check()
    assert all(g.pool.in_use == 0 for g in llm.cache.groups)


def test_searches_refused(on_cpu):
    from pico_vllm_b200 import BeamParams
    for bad in (dict(beams=0), dict(beams=33), dict(max_new_tokens=0), dict(length_penalty=-1.0), dict(length_penalty=float("nan")),
                dict(num_return=5), dict(num_return=0)):
        with pytest.raises(ConfigError):
            BeamParams(**bad)
    llm = beam_models.llm("qwen2/a", "cpu", 2, at_once=1, max_cache_tokens=96)
    with pytest.raises(ConfigError, match="slots"):
        llm.beam_search([[1, 2]], BeamParams(beams=3))
    with pytest.raises(ScheduleError, match="longest"):
        llm.beam_search([[1] * 90], BeamParams(beams=2, max_new_tokens=7))
    with pytest.raises(ScheduleError, match="at least one"):
        llm.beam_search([[]], BeamParams(beams=2))
    with pytest.raises(ConfigError, match="token ids"):
        llm.beam_search([[256]], BeamParams(beams=2))
    # six pages of 16: two beams of 80 tokens that share 2 pages at most do not fit, and everything comes back
    with pytest.raises(OutOfPages):
        llm.beam_search(beam_models.prompts_of("qwen2/a", (33,)), BeamParams(beams=2, max_new_tokens=60, ignore_eos=True))
    llm.cache.check()
    assert llm.cache.groups[0].pool.in_use == 0 and llm.cache.free_slots == 2
    assert len(llm.beam_search([[1, 2]], BeamParams(beams=2, max_new_tokens=3))[0].hypotheses) == 2


def test_a_vocabulary_smaller_than_the_beams(on_cpu):
    """Places that hold nothing go along without a trace: two tokens, five beams."""
    import fake_beam_ops as fake
    scores = torch.zeros(1, 1)
    tokens, parents, new, ended = fake.beam_select(torch.tensor([[0.0, 1.0]]), scores, 5, 1)
    assert tokens.tolist() == [[0, -1, -1, -1, -1]] and parents.tolist() == [[0, 1, 2, 3, 4]] and ended[0, 0] > -1
    assert new[0, 1:].tolist() == [-float("inf")] * 4
