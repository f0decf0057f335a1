"""Scratch of the linear cross entropy, whose kernels hand values to each other
through it: each call's own, also where two host threads enqueue on one stream
(the C call gives up the interpreter's lock) and where a graph has recorded it.
"""

import contextlib
import threading

import pytest
import torch

import tilec
from tilec import training


def test_calls_at_the_same_time_share_no_scratch(monkeypatch):
    # The host code alone, on CPU tensors: both calls are inside the library
    # before either returns.
    both = threading.Barrier(2, timeout=20)
    seen = []

    class Library:
        @staticmethod
        def tilec_linear_ce(*args):
            seen.append((args[18], args[19]))  # workspace, workspace_bytes
            if len(seen) > 1:  # after the first call
                both.wait()
            return 0

    monkeypatch.setattr(training._lib, "lib", lambda: Library)
    monkeypatch.setattr(training, "_on_gpu", lambda *a: 0)
    monkeypatch.setattr(training, "_on", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(training, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(training, "_ce_plan", lambda *a: (4096, 0, None))
    x, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    tilec.ext.linear_cross_entropy_grad(x, w, t)  # what is kept between calls is there
    threads = [threading.Thread(target=tilec.ext.linear_cross_entropy_grad, args=(x, w, t)) for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    _, (a, n), (b, m) = seen
    assert n == m == 4096 and (a + n <= b or b + m <= a)


def make(N, H, V, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(N, H, generator=g).to(dt).cuda(), (torch.randn(V, H, generator=g) * 0.1).to(dt).cuda(),
            torch.randint(V, (N,), generator=g).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_two_threads_on_one_stream(dt):
    f = tilec.ext.linear_cross_entropy_grad
    inputs = [make(200, 128, 3000, dt, 1), make(150, 192, 2000, dt, 2)]
    want = [f(*i) for i in inputs]
    got = [[], []]
    start = threading.Barrier(2, timeout=20)

    def work(k):
        start.wait()
        got[k] = [f(*inputs[k]) for _ in range(100)]

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    for k in range(2):
        assert len(got[k]) == 100
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(want[k], out))


def replay_after_a_larger_call(call, small, large):
    """A graph of call(small), replayed after call(large) on the stream it was
    recorded on and with all memory that was free then filled."""
    want = call(*small)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*small)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call(*small)
    with torch.cuda.stream(side):
        call(*large)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            filled = [torch.full((1 << k,), 0x55, dtype=torch.uint8, device="cuda") for k in range(9, 27) for _ in range(4)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))
        assert all((f == 0x55).all() for f in filled)
        del filled


@pytest.mark.gpu
def test_graph_after_a_larger_call():
    bf16 = torch.bfloat16
    replay_after_a_larger_call(tilec.ext.linear_cross_entropy_grad, make(40, 128, 1000, bf16, 3),
                               make(2000, 256, 6000, bf16, 4))
