"""The operators of 8-bit linear layers together, as a training step and a serving
step use them: against the same layer in plain float64 on the values that the codes
stand for, in captured graphs, and from two host threads."""

import math
import threading

import pytest
import torch

import tilec

F8 = torch.float8_e4m3fn
E32 = 2.0 ** -24


def make(R, D, H, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    return {"x": normal(R, D).bfloat16(), "res": normal(R, D, std=2.0).bfloat16(), "w": (1 + normal(D, std=0.1)).bfloat16(),
            "W": normal(H, D, std=1 / math.sqrt(D)), "dy": normal(R, H).bfloat16(), "dh": normal(R, D).bfloat16()}


def step(t, p, m, v):
    """Norm, product, its two gradients, the norm's gradients, clipping, optimizer."""
    x8, h, rstd = tilec.ext.rms_norm(t["x"], t["w"], t["res"], dtype=F8)
    W8 = tilec.ext.quantize_fp8(p, (128, 128))
    y = tilec.ext.linear_fp8(x8, W8, dtype=torch.bfloat16)
    dy = t["dy"]
    dn = tilec.ext.linear_fp8(tilec.ext.quantize_fp8(dy, dtype=torch.float8_e5m2), tilec.ext.quantize_fp8(p.t(), (128, 128)),
                              dtype=torch.bfloat16)
    n = tilec.ext.dequantize_fp8(x8, torch.bfloat16)
    dW = tilec.ext.linear_fp8(tilec.ext.quantize_fp8(dy.t(), dtype=torch.float8_e5m2), tilec.ext.quantize_fp8(n.t()))
    dx, dw = tilec.ext.rms_norm_backward(dn, h, rstd, t["w"], dh=t["dh"])
    norm, scale = tilec.ext.grad_norm([dW, dw], 1.0)
    tilec.ext.adamw_step([p], [dW], [m], [v], step=3, grad_scale=scale)
    return y, dx, dw, dW, norm, scale


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,H", [(1, 256, 128), (9, 300, 130), (200, 384, 257), (700, 1024, 640)])
def test_one_step_against_float64(R, D, H):
    # Rounding a value to e4m3 is off by 2^-4 of it at most, to e5m2 by 2^-3, and
    # uniformly so: about 0.6 of those in 2-norm (a third of the square), less what
    # mantissas vary.  A product's relative error is that of its operands, joined.
    t = make(R, D, H, R)
    p = t["W"].clone()
    y, dx, dw, dW, norm, scale = step(t, p, *tilec.ext.adamw_state(p))
    h = (t["x"].float() + t["res"].float()).bfloat16().double().requires_grad_()
    w, W = t["w"].double().requires_grad_(), t["W"].double().requires_grad_()
    n = h * (h.square().mean(dim=1, keepdim=True) + 1e-5) ** -0.5 * w
    want = n @ W.t()
    (want * t["dy"].double()).sum().backward()
    wdx = h.grad + t["dh"].double()

    def off(a, b):
        return ((a.double() - b).norm() / b.norm()).item()

    e4, e5 = 2.0 ** -4, 2.0 ** -3
    assert off(y, want) <= math.hypot(e4, e4) + 2.0 ** -8
    assert off(dW, W.grad) <= math.hypot(e5, e4) + 2.0 ** -8 + e4  # (n is rounded twice)
    assert off(dx, wdx) <= math.hypot(e5, e4) + 2.0 ** -8
    assert off(dw, w.grad) <= math.hypot(e5, e4) + 2.0 ** -8
    total = math.sqrt(float(dW.double().square().sum() + dw.double().square().sum()))
    assert abs(norm.item() - total) <= 4 * E32 * total
    assert abs(scale.item() - min(1.0, 1 / (total + 1e-6))) <= 4 * E32


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,H", [(1, 512, 640), (300, 384, 520)])
def test_graph_replays(R, D, H):
    # The whole step in one graph, replayed on new inputs with eager work in between;
    # every replay against the eager calls on the same inputs.
    t = make(R, D, H)
    p = t["W"].clone()
    m, v = tilec.ext.adamw_state(p)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(t, p, m, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(t, p, m, v)
    for k in range(4):
        new = make(R, D, H, seed=k + 1)
        for name in t:
            t[name].copy_(new[name])
        p.copy_(new["W"])
        m.zero_(), v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in (*out, p, m, v)]
        q = new["W"].clone()
        m2, v2 = tilec.ext.adamw_state(q)
        want = (*step(new, q, m2, v2), q, m2, v2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


@pytest.mark.gpu
def test_graphs_of_one_stream_at_the_same_time():
    # Two graphs captured on one stream, replayed on two, beside eager calls on the
    # stream they were captured on: each has a counter and scratch of its own.
    g = torch.Generator(device="cuda").manual_seed(0)
    lists = [[torch.randn(200000, generator=g, device="cuda") * s for _ in range(20)] for s in (1.0, 2.0, 3.0)]
    want = [[v.clone() for v in tilec.ext.grad_norm(l, 1.0)] for l in lists]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        tilec.ext.grad_norm(lists[0], 1.0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for l in lists[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append([tilec.ext.grad_norm(l, 1.0) for _ in range(10)])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(side):
            eager = [tilec.ext.grad_norm(lists[2], 1.0) for _ in range(10)]
        torch.cuda.synchronize()
        for got, ref in zip((*outs, eager), want):
            assert all(torch.equal(a, ref[0]) and torch.equal(b, ref[1]) for a, b in got)


@pytest.mark.gpu
def test_two_threads_on_one_stream():
    t = make(300, 500, 260)
    W8 = tilec.ext.quantize_fp8(t["W"], (128, 128))
    wide = torch.empty((260, 517), dtype=torch.uint8, device="cuda")  # rows that have to be copied
    wide[:, 3:503] = W8[0].view(torch.uint8)
    Wv = (wide.view(F8)[:, 3:503], W8[1])
    x8 = tilec.ext.quantize_fp8(t["x"])
    grads = [t["W"], t["dy"]]
    want = (tilec.ext.linear_fp8(x8, W8), *tilec.ext.grad_norm(grads, 1.0))
    torch.cuda.synchronize()
    bad = []

    def work():
        for _ in range(100):
            got = (tilec.ext.linear_fp8(x8, Wv), *tilec.ext.grad_norm(grads, 1.0))
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


def split_operands(M, N, K):
    g = torch.Generator().manual_seed(M + N)
    return tuple(tilec.ext.quantize_fp8(torch.randn(r, K, generator=g).cuda()) for r in (M, N))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_split_products_on_two_streams_and_in_graphs(dt):
    # Workgroups that share a tile count themselves in: counts of two streams, of a
    # graph and of the stream that it was recorded on are apart, and zero afterwards.
    f = tilec.ext.linear_fp8
    operands = [split_operands(*s) for s in ((70, 192, 9088), (38, 3584, 4800), (300, 100, 3000))]
    want = [f(*o, dtype=dt) for o in operands]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        inside = [f(*o, dtype=dt) for o in operands]
    for _ in range(4):
        out = []
        for s in streams[:2]:
            with torch.cuda.stream(s):
                out.append([f(*o, dtype=dt) for _ in range(5) for o in operands])
        with torch.cuda.stream(streams[2]):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i % 3]) for got in out for i, o in enumerate(got))
        assert all(torch.equal(o, w) for o, w in zip(inside, want))
        for o in inside:
            o.zero_()


@pytest.mark.gpu
def test_split_products_of_two_threads_on_one_stream():
    f = tilec.ext.linear_fp8
    operands = [split_operands(*s) for s in ((70, 192, 9088), (33, 4096, 2048))]
    want = [f(*o) for o in operands]
    got = [[], []]
    start = threading.Barrier(2, timeout=20)

    def work(k):
        start.wait()
        got[k] = [f(*operands[k]) for _ in range(100)]

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert all(len(g) == 100 and all(torch.equal(o, w) for o in g) for g, w in zip(got, want))
