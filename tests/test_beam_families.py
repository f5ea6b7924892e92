"""Families of the cache as large as they may be, and larger."""
import pytest
import torch

from pico_vllm_b200.cache import CacheManager
from pico_vllm_b200.errors import KernelError, PicoError
from test_beam_search import FULL, STATES, WIN, _Told, on_cpu  # noqa: F401  (a fixture)


def _family(entries, members):
    m = CacheManager(list(entries), 4, 200, members + 1, 80, torch.float32, "cpu", poison_freed=True)
    told = _Told(m)
    slot = m.acquire("r")
    told.write(slot, 6)
    line = [slot] + m.fork(slot, members - 1)
    for s in line[1:]:
        told.text[s] = list(told.text[slot])
    for s in line:
        told.write(s, 3)
    return m, told, line


def _limited(monkeypatch):
    """The doubles take as many places as the kernel does."""
    import pico_vllm_b200.ops as ops
    free = ops.reorder_states

    def limited(states, slots, parents):
        if slots.shape[1] > 32:
            raise KernelError("1 to 32 places")
        return free(states, slots, parents)
    monkeypatch.setattr(ops, "reorder_states", limited)


def test_a_family_too_large_for_its_states_is_refused_before_pages_move(on_cpu, monkeypatch):  # noqa: F811
    _limited(monkeypatch)
    m, told, line = _family((FULL, WIN) + STATES, 33)
    tables = [g.tables.copy() for g in m.groups]
    with pytest.raises(PicoError, match="32 at most"):
        m.reorder([line], [[1] * 33])
    assert all((g.tables == t).all() for g, t in zip(m.groups, tables))
    told.check()
    m.reorder([line], [list(range(33))])            # nothing moves
    m.reorder([line[:32]], [[31] + list(range(31))])
    texts = [told.text[s] for s in line[:32]]
    told.text.update({s: texts[q] for s, q in zip(line, [31] + list(range(31)))})
    told.check()


def test_families_without_states_may_be_larger(on_cpu, monkeypatch):  # noqa: F811
    _limited(monkeypatch)
    m, told, line = _family((FULL, WIN), 40)
    texts = [told.text[s] for s in line]
    parents = [(p * 7) // 10 for p in range(40)]
    m.reorder([line], [parents])
    told.text.update({s: list(texts[q]) for s, q in zip(line, parents)})
    told.check()
