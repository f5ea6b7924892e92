"""Host threads that call the same operator at the same time, each on a stream of its own."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def together(jobs):
    """Runs the jobs in threads that start together; what one of them raises is raised here."""
    start, failed = threading.Barrier(len(jobs)), []

    def go(job):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                job()
                torch.cuda.current_stream().synchronize()
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=go, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


def test_choices_of_different_sizes():
    """The lists of the two choices take 88 and 58 KB of a block's shared memory: both more than a kernel has without being asked for."""
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(7)
    inputs = [((torch.randn(rows, V, generator=g) * 3).to(DEV), (-torch.rand(1, rows, generator=g) * 5).to(DEV), rows) for rows, V in ((32, 9001), (16, 70000))]
    want = [[t.clone() for t in ops.beam_select(x, s, rows, 3)] for x, s, rows in inputs]
    torch.cuda.synchronize()

    def job(k):
        x, s, rows = inputs[k]
        for i in range(3000):
            got = ops.beam_select(x, s, rows, 3)
            if i % 500 == 0:
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want[k]))
    together([lambda: job(0), lambda: job(1), lambda: job(0)])


def test_router_and_norms_of_different_widths():
    """Kernels whose rows lie in shared memory take more of it for wider rows."""
    from pico_vllm_b200 import ops
    g = torch.Generator().manual_seed(8)

    def routing(width):
        h, w = torch.randn(6, width, generator=g).to(DEV), (torch.randn(64, width, generator=g) / width ** 0.5).to(DEV)
        return lambda: ops.moe_route(h, w, None, 4)

    def norm(width):
        x, w = torch.randn(5, width, generator=g).to(DEV), torch.randn(width, generator=g).to(DEV)
        return lambda: (ops.add_rmsnorm(x, None, w, 1e-6, torch.empty_like(x)),)
    calls = [make(width) for make in (routing, norm) for width in (14000, 20000)]
    want = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()

    def job(k):
        for i in range(2000):
            for c in (k, 2 + k):
                r = calls[c]()
                if i % 500 == 0:
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(r, want[c]))
    together([lambda: job(0), lambda: job(1), lambda: job(0)])
