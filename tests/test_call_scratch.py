"""Scratch of the linear cross entropy, whose kernels hand values to each other
through it: each call's own, also where two host threads enqueue on one stream
(the C call gives up the interpreter's lock) and where a graph has recorded it.
And the buffers that products and sums on a stream share, where a graph has
recorded them and where two host threads use them.
"""

import contextlib
import gc
import threading
import time
import weakref

import pytest
import torch

import tilec
from tilec import ext, training


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


@pytest.mark.parametrize("get", [ext.workspace_for, ext.counters_for])
def test_buffers_and_captures(monkeypatch, get):
    # The host code alone, on CPU memory: what a capture used outlives a larger
    # call, and what a capture allocated (zeroed only when the graph runs) does
    # not reach the calls after it.
    now = [False]
    monkeypatch.setattr(ext, "_capturing", lambda device: now[0], raising=False)
    cpu, stream = torch.device("cpu"), 987654321
    now[0] = True
    inside = get(cpu, stream, 100)
    now[0] = False
    eager = get(cpu, stream, 100)
    assert eager.data_ptr() != inside.data_ptr() and get(cpu, stream, 50) is eager
    now[0] = True
    assert get(cpu, stream, 100) is eager
    larger = get(cpu, stream, 5 << 20)
    assert larger.numel() >= 5 << 20 and get(cpu, stream, 100) is eager
    now[0] = False
    recorded = weakref.ref(eager.untyped_storage())
    eager = None
    assert get(cpu, stream, 6 << 20).numel() >= 6 << 20
    gc.collect()
    assert recorded() is not None
    unrecorded = weakref.ref(get(cpu, stream, 100).untyped_storage())
    get(cpu, stream, 7 << 20)
    gc.collect()
    assert unrecorded() is None


def test_counters_outlive_the_call_they_are_for(monkeypatch):
    # The host code alone, on CPU tensors: another thread's call that needs more
    # counters replaces the buffer while this call is inside the library.
    held = []

    class Library:
        @staticmethod
        def tilec_linear_ce(*args):
            buffer = weakref.ref(ext._COUNTERS[None, 987654319].untyped_storage())
            ext.counters_for(torch.device("cpu"), 987654319, 1 << 20)
            gc.collect()
            held.append(buffer() is not None)
            return 0

    monkeypatch.setattr(training._lib, "lib", lambda: Library)
    monkeypatch.setattr(training, "_on_gpu", lambda *a: 0)
    monkeypatch.setattr(training, "_on", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(training, "_raw_stream", lambda index: 987654319)
    monkeypatch.setattr(training, "_ce_plan", lambda *a: (4096, 256, None))
    x, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    tilec.ext.linear_cross_entropy_grad(x, w, t)
    assert held == [True]


def test_products_that_share_scratch_are_enqueued_one_by_one(monkeypatch):
    # The host code alone, on CPU tensors: while one call is inside the library
    # another does not get there.
    inside, most = [], []

    class Library:
        @staticmethod
        def tilec_matmul(*args):
            inside.append(args[13])
            most.append(len(inside))
            time.sleep(0.05)
            inside.pop()
            return 0

    monkeypatch.setattr(ext._lib, "lib", lambda: Library)
    monkeypatch.setattr(ext, "_raw_stream", lambda device: 987654320)
    monkeypatch.setattr(ext, "_scratch_sizes", lambda *a: (4096, 64))
    x = torch.zeros(8, 8)
    threads = [threading.Thread(target=ext._launch, args=(x, x, 8, 8, 8, 0, 1)) for _ in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert most == [1, 1, 1]


def test_a_product_in_a_signal_handler_does_not_wait_for_the_call_it_interrupts(monkeypatch):
    # The host code alone: the handler runs while this thread's call is being
    # enqueued.
    calls = []

    class Library:
        @staticmethod
        def tilec_matmul(*args):
            calls.append(args[13])
            if len(calls) == 1:  # what a handler would do here
                ext._launch(x, x, 8, 8, 8, 0, 1)
            return 0

    monkeypatch.setattr(ext._lib, "lib", lambda: Library)
    monkeypatch.setattr(ext, "_raw_stream", lambda index: 987654318)
    monkeypatch.setattr(ext, "_scratch_sizes", lambda *a: (4096, 64))
    x = torch.zeros(8, 8)
    outer = threading.Thread(target=ext._launch, args=(x, x, 8, 8, 8, 0, 1), daemon=True)
    outer.start()
    outer.join(timeout=10)
    assert not outer.is_alive() and len(calls) == 2


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


@pytest.mark.gpu
def test_two_threads_copy_operands_on_one_stream():
    # Variants that copy unaligned operands into the scratch first.
    variant = next(v["name"] for v in tilec._lib.variants() if v["dtype"] == tilec._lib.BF16 and ext.pad_variant(v))
    inputs = [(make(201, 333, 257, torch.bfloat16, s)[:2]) for s in (8, 9)]
    inputs = [(x, w.t()) for x, w in inputs]
    want = [ext.matrix_mul(*i, variant) for i in inputs]
    got = [[], []]
    start = threading.Barrier(2, timeout=20)

    def work(k):
        start.wait()
        got[k] = [ext.matrix_mul(*inputs[k], variant) for _ in range(200)]

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert all(len(g) == 200 and all(torch.equal(out, w) for out in g) for g, w in zip(got, want))


def replay_after_a_larger_call(call, small, large, replaced=()):
    """A graph of call(small), replayed after call(large) on the stream it was
    recorded on and with all memory that was free then filled.  `replaced`:
    tables of ext whose buffer of that stream call(large) replaces."""
    want = call(*small)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*small)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call(*small)
    key = (torch.cuda.current_device(), side.cuda_stream)
    before = [table[key].data_ptr() for table in replaced]
    with torch.cuda.stream(side):
        call(*large)
    torch.cuda.synchronize()
    assert all(table[key].data_ptr() != p for table, p in zip(replaced, before))
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


@pytest.mark.gpu
def test_graph_of_split_products_after_a_larger_call():
    # Products and sums that split K, and the float32 loss, whose products may:
    # their counters have to be there, and zero, at every replay.
    variant = next(v["name"] for v in tilec._lib.variants()
                   if v["dtype"] == tilec._lib.F32 and v["family"] == tilec._lib.FAMILY_SKINNY and not ext.rows_variant(v))

    def call(x, w, t):
        return (ext.matrix_mul(x, w.t().contiguous(), (variant, 8)), ext.sum(x), *ext.linear_cross_entropy_grad(x, w, t))

    f32 = torch.float32
    small, large = make(4, 4096, 64, f32, 5), make(16, 4096, 30000, f32, 6)
    replay_after_a_larger_call(call, small, large, (ext._SCRATCH, ext._COUNTERS))


@pytest.mark.gpu
def test_graph_without_calls_before_it():
    x, w, t = make(4, 4096, 64, torch.float32, 7)
    variant = next(v["name"] for v in tilec._lib.variants()
                   if v["dtype"] == tilec._lib.F32 and v["family"] == tilec._lib.FAMILY_SKINNY and not ext.rows_variant(v))
    b = w.t().contiguous()

    def call():
        return ext.matrix_mul(x, b, (variant, 8)), ext.matrix_mul(x, b, (variant, 4))

    want = call()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    for _ in range(3):
        with torch.cuda.stream(side):
            eager = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)) and all(torch.equal(a, b) for a, b in zip(want, eager))
