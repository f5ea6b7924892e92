"""Rows of the cache that do not exist are told by check_kernel_status, whatever stream the call went to."""
import pytest
import torch

import plain_beam as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)


def _busy():
    """Some 50 ms of work before what follows on the current stream."""
    x = torch.randn(8192, 8192, device=DEV, dtype=torch.bfloat16)
    for _ in range(60):
        x = (x @ x) * 1e-2


def _calls(d):
    """A call of each kind with an index that is no row of d [2, 6, ...], its tensors made beforehand."""
    from pico_vllm_b200 import ops
    src, dst = torch.tensor([0, 6], **I32), torch.tensor([3, 4], **I32)
    slots, parents = torch.tensor([[0, 1, 9]], **I32), torch.tensor([[1, 0, 0]], **I32)
    return {"copy": lambda: ops.copy_pages([d], src, dst), "reorder": lambda: ops.reorder_states([d], slots, parents)}


def _after(t, kind):
    return plain.copy(t, [0], [3]) if kind == "copy" else plain.reorder(t, [[0, 1]], [[1, 0]])


@pytest.mark.parametrize("width", [40, 41])             # rows that lie on 16 bytes, rows that do not
@pytest.mark.parametrize("kind", ["copy", "reorder"])
def test_told_after_a_call_on_a_stream_of_its_own(kind, width):
    """The call is still waiting for its turn when the status is asked for on its stream; or on another one, where it is told once the call has run."""
    from pico_vllm_b200 import ops
    from pico_vllm_b200.errors import KernelError
    t = torch.randn(2, 6, width, generator=torch.Generator().manual_seed(1))
    d = t.to(DEV)
    call = _calls(d)[kind]
    none = torch.zeros(1, 1, **I32)
    ops.copy_pages([d], none[0], none[0])               # (loads the kernel: that would wait for the device)
    ops.reorder_states([d], none, none)
    ops.check_kernel_status()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        _busy()
        call()
        with pytest.raises(KernelError, match="outside a tensor"):
            ops.check_kernel_status()
        ops.check_kernel_status()                       # told once
    assert torch.equal(d.cpu(), _after(t, kind))
    for early in (True, False):
        with torch.cuda.stream(stream):
            _busy()
            call()
        told = ops.rows_status() if early else 0        # (mostly before the call has run)
        stream.synchronize()
        assert told + ops.rows_status() == 1 and ops.rows_status() == 0


def test_told_for_every_stream_and_every_replay():
    from pico_vllm_b200 import ops
    from pico_vllm_b200.errors import KernelError
    ds = [torch.randn(2, 6, 40, device=DEV) for _ in range(2)]
    calls = [_calls(d)["copy"] for d in ds]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for order in ((0, 1), (1, 0)):
        for k in order:
            with torch.cuda.stream(streams[k]):
                _busy()
                calls[k]()
        for k in order:
            with torch.cuda.stream(streams[k]):
                ops.rows_status()                       # 1 at least once
        assert ops.rows_status() == 0
        with torch.cuda.stream(streams[order[0]]):
            calls[order[0]]()
            assert ops.rows_status() == 1 and ops.rows_status() == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls[0]()
        assert ops.rows_status() == 0                   # (a stream that is being recorded is not asked)
    ops.check_kernel_status()                           # (recorded, not run)
    for _ in range(3):
        graph.replay()
        with pytest.raises(KernelError, match="outside a tensor"):
            ops.check_kernel_status()
        ops.check_kernel_status()


def test_more_tensors_than_a_launch_takes_are_told_once():
    """Tensors with different numbers of rows, in three launches: what is a row of one is none of another."""
    from pico_vllm_b200 import ops
    from pico_vllm_b200.errors import KernelError
    g = torch.Generator().manual_seed(2)
    ts = [torch.randn(2, 4 + k % 3, 8 + k % 5, generator=g) for k in range(37)]
    ds = [t.to(DEV) for t in ts]
    ops.copy_pages(ds, torch.tensor([1, 5], **I32), torch.tensor([3, 0], **I32))
    with pytest.raises(KernelError, match="outside a tensor"):
        ops.check_kernel_status()
    ops.check_kernel_status()
    for t, d in zip(ts, ds):
        assert torch.equal(d.cpu(), plain.copy(t, [1] + [5] * (t.shape[1] > 5), [3] + [0] * (t.shape[1] > 5)))


def test_asking_does_not_end_a_recording_of_another_thread():
    """A thread records calls while another one asks, again and again."""
    import threading
    from pico_vllm_b200 import ops
    t = torch.randn(2, 6, 40, device=DEV)
    pairs = torch.tensor([[0], [3]], **I32)
    ops.copy_pages([t], pairs[0], pairs[1])
    ops.check_kernel_status()
    torch.cuda.synchronize()
    recording, asked, failed = threading.Event(), threading.Event(), []

    def record():
        try:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, capture_error_mode="thread_local"):
                ops.copy_pages([t], pairs[0], pairs[1])
                recording.set()
                asked.wait(20)
                ops.copy_pages([t], pairs[0], pairs[1])
            graph.replay()
            torch.cuda.synchronize()
        except BaseException as e:
            failed.append(e)
            recording.set()
    thread = threading.Thread(target=record)
    thread.start()
    recording.wait(20)
    try:
        assert not failed
        for _ in range(20):
            ops.check_kernel_status()
    finally:
        asked.set()
        thread.join()
    assert not failed, failed
    assert torch.equal(t[:, 0], t[:, 3])
