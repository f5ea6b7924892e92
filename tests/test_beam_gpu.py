"""The kernels of beam search against plain computations: the choice of beams in float64, rows of the cache moved one by one."""
import math
import random

import pytest
import torch

import plain_beam as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ------------------------------------------------------------------ the choice
def _logits(kind, rows, V, g):
    x = torch.randn(rows, V, generator=g) * 2.0
    if kind == "peaks":
        x.scatter_(1, torch.randint(0, V, (rows, min(V, 30)), generator=g), 9.0)
        x += torch.randn(rows, V, generator=g) * 0.3
    elif kind == "equal":                  # one number everywhere: the first tokens of the first beam
        x.fill_(0.25)
    elif kind == "steps":                  # few values: ties by the dozen, the same ones in every beam
        x = torch.randint(-3, 4, (1, V), generator=g).float().repeat(rows, 1)
    elif kind == "zeros":                  # 0 and -0 are one value
        x = torch.where(torch.rand(rows, V, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "rising":
        x = torch.linspace(-20, 11, V).repeat(rows, 1) + torch.arange(rows)[:, None] * 1e-2
    elif kind == "falling":
        x = torch.linspace(11, -20, V).repeat(rows, 1) + torch.arange(rows)[:, None] * 1e-2
    elif kind == "crowded":                # all that counts lies side by side
        x[:, V // 3:V // 3 + 200] += 15.0
    elif kind == "masked":
        x[torch.rand(rows, V, generator=g) < 0.97] = -math.inf
    elif kind == "lowest":                 # masked by the type's lowest number
        x[torch.rand(rows, V, generator=g) < 0.97] = torch.finfo(torch.float32).min
    elif kind == "huge":
        x *= 1e37
    elif kind == "odd rows":               # one masked whole, one with NaN, one with an infinity, if there are as many
        x[0] = -math.inf
        if rows > 1:
            x[1, V // 2] = math.nan
        if rows > 2:
            x[2, V - 1] = math.inf
    return x


def _check(logits, scores, beams, end, got, G, rows, V):
    tokens, parents, new, ended = (t.cpu() for t in got)
    # A value's error: that of the normaliser - sums of 16 exponentials and then of tiles, parts and threads in 32 bits (at most one rounding
    # a term, 2^-24 of the sum each), exponentials off by 2^-22 and by 2^-23 of the distance (taken as 64 at most: terms beyond do not count) -
    # and the rounding of the result
    off = (V / 4096 + 16 + 16) * 2.0 ** -24 + 2.0 ** -22 + 64 * 2.0 ** -23
    for g in range(G):
        x, s = logits[g * rows:(g + 1) * rows], scores[g]
        wt, wp, ws, we, ranked = plain.select(x, s, beams, end)
        # candidates of different beams are compared by values that the kernel has to within `off`: equal ones (beams that are the same) or far apart
        assert all(a[0] == b[0] or a[1] == b[1] or a[0] - b[0] > 2 * off for a, b in zip(ranked, ranked[1:])), "inputs too near a tie"
        assert tokens[g].tolist() == wt and parents[g].tolist() == wp, g
        for a, b in zip(new[g].tolist() + ended[g].tolist(), ws + we):
            if math.isinf(b):
                assert a == b
            else:
                assert abs(a - b) <= off + abs(b) * 2.0 ** -24, (a, b)


SIZES = [(1, 1, 1, 1), (1, 1, 4, 2), (2, 3, 3, 5), (3, 4, 4, 257), (2, 1, 8, 4096), (5, 2, 5, 4097), (1, 4, 4, 151936), (2, 32, 32, 9001),
         (1, 32, 32, 20000), (2, 20, 20, 30001), (1, 2, 32, 30000), (40, 4, 4, 33001), (1, 1, 32, 70000), (3, 7, 19, 12289)]


@pytest.mark.parametrize("G,rows,beams,V", SIZES)
@pytest.mark.parametrize("kind", ["bell", "peaks", "equal", "steps", "zeros", "rising", "falling", "crowded", "masked", "lowest", "huge", "odd rows"])
def test_choice_of_beams(G, rows, beams, V, kind):
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(1000 * G + 10 * beams + V)
    logits = torch.cat([_logits(kind, rows, V, g) for _ in range(G)])
    # scores some way apart, so that candidates of different beams are no nearer than chance makes them; the same where ties are the point
    scores = -torch.rand(G, rows, generator=g) * 5 - 3
    if kind in ("equal", "steps", "zeros"):
        scores[:] = -2.5
    if rows > 2:
        scores[0, rows - 1] = -math.inf
    logits, scores = logits.to(DEV), scores.to(DEV)
    wide = torch.empty(G * rows, V + 3, device=DEV)
    wide[:, 1:1 + V] = logits
    for end in (None, V // 2, int(logits[0].nan_to_num(-math.inf).argmax())):
        got = ops.beam_select(logits, scores, beams, end)
        _check(logits, scores, beams, end, got, G, rows, V)
        for a, b in zip(got, ops.beam_select(wide[:, 1:1 + V], scores, beams, end)):      # rows that start on any 4 bytes: the same sums
            assert torch.equal(a, b)
    ops.check_kernel_status()


def test_scores_not_numbers_and_one_row_for_all():
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(5)
    row = torch.randn(1, 5000, generator=g)
    scores = torch.tensor([[-1.0, math.nan, math.inf, -math.inf], [-math.inf] * 4])
    got = ops.beam_select(row.to(DEV).expand(8, 5000), scores.to(DEV), 4, 7)
    _check(row.repeat(8, 1), scores, 4, 7, got, 2, 4, 5000)
    assert got[0][1].tolist() == [-1] * 4 and got[1][1].tolist() == [0, 1, 2, 3]


def test_choice_into_a_buffer_step_after_step_and_recorded():
    """The scores of a step are where the step before left them; a recorded step gives what a direct one does, twice."""
    from pico_vllm_b200 import ops
    G, B, V = 3, 4, 9999
    g = torch.Generator().manual_seed(9)
    steps = [(torch.randn(G * B, V, generator=g) * 3).to(DEV) for _ in range(3)]
    first = (-torch.rand(G, B, generator=g)).to(DEV)

    def direct():
        scores, seen = first, []
        for x in steps:
            r = ops.beam_select(x, scores, B, 11)
            scores = r[2].clone()
            seen.append([t.clone() for t in r])
        return seen
    want = direct()
    out = torch.empty(G * 4 * B, dtype=torch.int32, device=DEV)
    x, scores = torch.empty_like(steps[0]), torch.empty_like(first)
    ops.beam_select(steps[0], first, B, 11, out)
    held = out[2 * G * B:3 * G * B].view(torch.float32).view(G, B)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.beam_select(x, held, B, 11, out)
    for _ in range(2):
        held.copy_(first)
        for step, w in zip(steps, want):
            x.copy_(step)
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_two_streams_at_once():
    from pico_vllm_b200 import ops
    G, B, V = 4, 4, 50001
    g = torch.Generator().manual_seed(4)
    jobs = [((torch.randn(G * B, V, generator=g) * 3).to(DEV), (-torch.rand(G, B, generator=g)).to(DEV)) for _ in range(2)]
    want = [[t.clone() for t in ops.beam_select(x, s, B, 3)] for x, s in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for k, (x, s) in enumerate(jobs):
            with torch.cuda.stream(streams[k]):
                got[k].append(ops.beam_select(x, s, B, 3))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for r in got[k] for a, b in zip(r, want[k]))


# ------------------------------------------------------------------ rows
def _random_tensor(shape, dtype, g):
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g).to(dtype)
    return torch.randint(0, 100, shape, generator=g).to(dtype)


ROWS = [((3, 40, 16, 8), torch.float32), ((1, 33, 7, 97), torch.bfloat16), ((2, 40, 5), torch.uint8), ((5, 35, 1), torch.int64), ((2, 36, 129, 128), torch.float32),
        ((4, 34), torch.float32), ((2, 40, 3), torch.bfloat16), ((3, 40, 37), torch.uint8), ((2, 33, 4099), torch.uint8), ((1, 34, 1001, 3), torch.float32)]


def _views(t):
    """The tensor as it is, as every second row of a longer one that starts an element later, and with rows outside entries."""
    E, N = t.shape[:2]
    yield t.to(DEV)
    rest = t[0, 0].numel()
    flat = torch.empty(1 + E * 2 * N * rest, dtype=t.dtype, device=DEV)
    v = flat[1:].view(E, 2 * N, *t.shape[2:])[:, ::2]
    v.copy_(t)
    yield v
    yield t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)


@pytest.mark.parametrize("shape,dtype", ROWS)
def test_pages_copied(shape, dtype):
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(shape[1])
    t = _random_tensor(shape, dtype, g)
    order = torch.randperm(shape[1], generator=g).tolist()
    src, dst = order[:12], order[12:22] + [-1, order[11]]        # a pair for padding, one with itself
    src[9] = -3
    want = plain.copy(t, src, dst)
    for v in _views(t):
        other = v.clone()
        ops.copy_pages([v, other], torch.tensor(src, dtype=torch.int32, device=DEV), torch.tensor(dst, dtype=torch.int32, device=DEV))
        assert torch.equal(v.cpu(), want) and torch.equal(other.cpu(), want)
    ops.check_kernel_status()


@pytest.mark.parametrize("shape,dtype", ROWS)
@pytest.mark.parametrize("places", [1, 2, 3, 4, 8, 11, 32])
def test_states_passed_on(shape, dtype, places):
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(places)
    rng = random.Random(places)
    t = _random_tensor(shape, dtype, g)
    G = shape[1] // places
    slots = torch.randperm(shape[1], generator=g)[:G * places].view(G, places).tolist()
    families = {
        "any": [[rng.randrange(places) for _ in range(places)] for _ in range(G)],
        "cycles": [torch.randperm(places, generator=g).tolist() for _ in range(G)],
        "one round": [[(p + 1) % places for p in range(places)] for _ in range(G)],
        "pairs": [[min(p ^ 1, places - 1) for p in range(places)] for _ in range(G)],
        "one parent": [[places - 1] * places for _ in range(G)],
        "none": [list(range(places)) for _ in range(G)],
    }
    for parents in families.values():
        want = plain.reorder(t, slots, parents)
        for v in _views(t):
            other = v.clone()
            ops.reorder_states([v, other], torch.tensor(slots, dtype=torch.int32, device=DEV), torch.tensor(parents, dtype=torch.int32, device=DEV))
            assert torch.equal(v.cpu(), want) and torch.equal(other.cpu(), want)
    ops.check_kernel_status()


def test_more_tensors_than_a_launch_takes_and_none():
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(2)
    ts = [torch.randn(2, 9, 1 + k, generator=g) for k in range(37)] + [torch.empty(2, 9, 0), torch.empty(0, 9, 4)]
    dev = [t.to(DEV) for t in ts]
    i32 = dict(dtype=torch.int32, device=DEV)
    ops.copy_pages(dev, torch.tensor([1, 2], **i32), torch.tensor([5, 0], **i32))
    ops.reorder_states(dev, torch.tensor([[3, 4, 8]], **i32), torch.tensor([[1, 0, 0]], **i32))
    for t, d in zip(ts, dev):
        assert torch.equal(d.cpu(), plain.reorder(plain.copy(t, [1, 2], [5, 0]), [[3, 4, 8]], [[1, 0, 0]]))
    before = ops.launches
    ops.copy_pages([], torch.tensor([1], **i32), torch.tensor([2], **i32))
    ops.copy_pages(dev[:1], torch.empty(0, **i32), torch.empty(0, **i32))
    ops.reorder_states(dev[:1], torch.empty(0, 4, **i32), torch.empty(0, 4, **i32))
    assert ops.launches == before


def test_offsets_beyond_32_bits():
    from pico_vllm_b200 import ops
    i32 = dict(dtype=torch.int32, device=DEV)
    t = torch.zeros(2, 3, (1 << 30) + 16, dtype=torch.uint8, device=DEV)           # 6.4 GB
    t[:, 0, ::4099] = 7
    t[:, 0, -1] = 9
    ops.copy_pages([t], torch.tensor([0], **i32), torch.tensor([2], **i32))
    assert torch.equal(t[0, 0], t[0, 2]) and torch.equal(t[1, 0], t[1, 2]) and int(t[:, 1].max()) == 0
    ops.reorder_states([t], torch.tensor([[1, 2]], **i32), torch.tensor([[1, 0]], **i32))
    assert torch.equal(t[1, 0], t[1, 1]) and torch.equal(t[0, 0], t[0, 1]) and int(t[:, 2].max()) == 0


def test_an_index_that_is_no_row_is_passed_over_and_told():
    from pico_vllm_b200 import ops
    from pico_vllm_b200.errors import KernelError
    i32 = dict(dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(3)
    t = torch.randn(2, 6, 40, generator=g)
    d = t.to(DEV)
    ops.copy_pages([d], torch.tensor([0, 6, 1], **i32), torch.tensor([3, 4, 2 ** 31 - 1], **i32))
    assert torch.equal(d.cpu(), plain.copy(t, [0], [3]))
    with pytest.raises(KernelError, match="outside a tensor"):
        ops.check_kernel_status()
    ops.check_kernel_status()                           # told once
    for slots, parents in (([[0, 1, 6]], [[1, 0, 0]]), ([[0, 1, 2]], [[1, 0, 3]]), ([[0, 1, 2]], [[1, 0, -1]]), ([[0, 1, -7]], [[1, 0, 0]])):
        d = t.to(DEV)
        ops.reorder_states([d], torch.tensor(slots, **i32), torch.tensor(parents, **i32))
        assert torch.equal(d.cpu(), plain.reorder(t, [[0, 1]], [[1, 0]]))
        with pytest.raises(KernelError, match="outside a tensor"):
            ops.check_kernel_status()


def test_rows_moved_in_a_recorded_call():
    from pico_vllm_b200 import ops
    i32 = dict(dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(8)
    t = torch.randn(3, 20, 50, generator=g)
    d = t.to(DEV)
    slots, parents = torch.tensor([[4, 5, 6], [1, 9, 0]], **i32), torch.tensor([[0, 1, 2], [0, 1, 2]], **i32)
    src, dst = torch.full((4,), -1, **i32), torch.full((4,), -1, **i32)
    ops.copy_pages([d], src, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reorder_states([d], slots, parents)
        ops.copy_pages([d], src, dst)
    for family, pairs in (([[2, 2, 1], [1, 2, 0]], [(4, 12)]), ([[0, 0, 0], [0, 1, 2]], [(1, 13), (9, 14)])):
        parents.copy_(torch.tensor(family))
        src.fill_(-1)
        dst.fill_(-1)
        for k, (s, e) in enumerate(pairs):
            src[k], dst[k] = s, e
        graph.replay()
        t = plain.copy(plain.reorder(t, slots.tolist(), family), [p[0] for p in pairs], [p[1] for p in pairs])
        assert torch.equal(d.cpu(), t)


def test_another_device_than_the_current_one_is_refused(monkeypatch):
    from pico_vllm_b200 import ops
    from pico_vllm_b200.errors import KernelError
    i32 = dict(dtype=torch.int32, device=DEV)
    x, s, t = torch.zeros(4, 8, device=DEV), torch.zeros(1, 4, device=DEV), torch.zeros(2, 3, 4, device=DEV)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: ops.beam_select(x, s, 4), lambda: ops.copy_pages([t], torch.zeros(1, **i32), torch.zeros(1, **i32)),
                 lambda: ops.reorder_states([t], torch.zeros(1, 2, **i32), torch.zeros(1, 2, **i32))):
        with pytest.raises(KernelError, match="current device"):
            call()


def test_on_a_stream_of_its_own():
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(6)
    t, x = torch.randn(3, 30, 5000, generator=g), torch.randn(8, 20001, generator=g) * 3
    scores = -torch.rand(2, 4, generator=g)
    slots, parents = [[3, 9, 1, 20], [5, 6, 7, 8]], [[1, 2, 0, 0], [0, 0, 2, 2]]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        big = torch.randn(4096, 4096, device=DEV)
        for _ in range(10):
            big = (big @ big) * 1e-2                   # what comes before is still under way when the calls are made
        d, lx = t.to(DEV, non_blocking=True), x.to(DEV, non_blocking=True)
        i32 = dict(dtype=torch.int32, device=DEV)
        ops.reorder_states([d], torch.tensor(slots, **i32), torch.tensor(parents, **i32))
        ops.copy_pages([d], torch.tensor([3, 5], **i32), torch.tensor([11, 12], **i32))
        got = ops.beam_select(lx, scores.to(DEV), 4, 5)
    stream.synchronize()
    assert torch.equal(d.cpu(), plain.copy(plain.reorder(t, slots, parents), [3, 5], [11, 12]))
    _check(x, scores, 4, 5, got, 2, 4, 20001)


def test_a_vocabulary_of_many_millions():
    """Offsets of bytes beyond 32 bits, and as many parts of a row as the join takes."""
    from pico_vllm_b200 import ops
    V = 150_000_003
    logits = torch.empty(8, V, device=DEV)[6:]             # (starts 3.6 GB into its memory)
    g = torch.Generator(device=DEV).manual_seed(12)
    logits.copy_(torch.randint(-30, 0, (2, V), generator=g, device=DEV))
    at = torch.randperm(V, generator=torch.Generator().manual_seed(1))[:9].tolist()
    for k, t in enumerate(at):
        logits[k % 2, t] = 20.0 + 0.25 * k
    scores = torch.tensor([[-1.0, -0.5]], device=DEV)
    got = ops.beam_select(logits, scores, 4, at[5])
    # what the two rows' sums are does not matter to the order here: the large ones differ by 0.25 and more, and so do the normalisers
    x = logits.double()
    lse = (x - x.amax(1, keepdim=True)).exp().sum(1).log() + x.amax(1)
    value = sorted(((20.0 + 0.25 * k - float(lse[k % 2]) + float(scores[0, k % 2]), k % 2, t) for k, t in enumerate(at)), reverse=True)
    assert all(a[0] - b[0] > 1e-3 for a, b in zip(value, value[1:]))
    want = [v for v in value if v[2] != at[5]][:4]
    tokens, parents, new, ended = (t.cpu() for t in got)
    assert sorted(zip(parents[0].tolist(), tokens[0].tolist())) == sorted((b, t) for _, b, t in want)
    # sums of up to 1.5e8 / (32 * 256 * 16) tiles of 16 terms a thread, 2^-24 of the sum for each at most
    for b, t, v in zip(parents[0].tolist(), tokens[0].tolist(), new[0].tolist()):
        assert abs(v - next(w[0] for w in want if w[1:] == (b, t))) <= (1200 + 64) * 2.0 ** -24 + 2.0 ** -17
    assert (ended[0, 1] > -math.inf) == ((at[5]) in [v[2] for v in value[:4]]) and ended[0, 0] == -math.inf


def test_a_buffer_that_overlaps_the_inputs_is_refused():
    from pico_vllm_b200 import ops
    from pico_vllm_b200.errors import KernelError
    memory = torch.zeros(4000, dtype=torch.int32, device=DEV)
    floats = memory.view(torch.float32)
    logits, scores, out = floats[:800].view(8, 100), floats[900:908].view(2, 4), memory[1000:1032]
    ops.beam_select(logits, scores, 4, None, out)
    ops.beam_select(logits, out[16:24].view(torch.float32).view(2, 4), 4, None, out)              # the new scores of before
    for at in (0, 768, 799, 876, 901, 907):
        with pytest.raises(KernelError, match="overlaps"):
            ops.beam_select(logits, scores, 4, None, memory[at:at + 32])
    ops.beam_select(logits, scores, 4, None, memory[800:832])
    with pytest.raises(KernelError, match="overlaps"):
        ops.beam_select(logits, out[15:23].view(torch.float32).view(2, 4), 4, None, out)
    with pytest.raises(KernelError, match="overlaps"):                                            # two rows for four beams: other places
        ops.beam_select(logits[:4], out[16:20].view(torch.float32).view(2, 2), 4, None, memory[1000:1028])
