"""AdamW steps over many tensors against a plain 64-bit form: types, sizes and
alignments, 32-bit and 8-bit states, special values and refusals.

Tolerances.  m and v are two products and a sum, each rounded once: 4 roundings
of the magnitudes added.  p adds to its own 3 roundings the error of the step
taken, rate |m / denom| times at most 12 roundings plus the relative error of m
where its terms cancel.  The value of a v code: 1 / 255 and its product with
the code are rounded (2 roundings), their square doubles that and adds one (5),
the fourth power again (11), the scale adds one: 12; of an m code: 6.  An 8-bit
code is at most half a code (and the roundings of its root and quotient, 1e-4 of
a code) from the exact one.
"""

import math

import pytest
import torch

import tilec

E32 = 2.0 ** -24
HYPER = {"lr": 3e-3, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.1}
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 70001]


def tensors(sizes, dtype, seed, std, lo=0):
    """Views of one storage that start at odd elements (lo + multiples of odd
    numbers), values N(0, std)."""
    g = torch.Generator().manual_seed(seed)
    room = sum(sizes) + 7 * len(sizes) + lo
    flat = (torch.randn(room, generator=g) * std).to(dtype).cuda()
    out, at = [], lo
    for n in sizes:
        out.append(flat[at:at + n])
        at += n + 7
    return out


def plain(p, g, m, v, step, lr, betas, eps, weight_decay, scale=1.0):
    """(p, m, v) of one step, and bounds of their errors."""
    b1, b2 = betas
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * scale
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    em = 5 * E32 * (b1 * m.abs() + (1 - b1) * g.abs())
    ev = 6 * E32 * v2
    denom = v2.sqrt() / math.sqrt(1 - b2 ** step) + eps
    rate = lr / (1 - b1 ** step)
    p2 = p * (1 - lr * weight_decay) - rate * m2 / denom
    ep = 4 * E32 * p.abs() + rate * (em / denom + 12 * E32 * (m2 / denom).abs())
    return (p2, m2, v2), (ep, em + 1e-44, ev + 1e-44)


def near(got, want, bound, extra=0.0):
    assert ((got.double() - want).abs() <= bound + extra * (want.abs() + bound) + 1e-44).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lo", [0, 1])
def test_states_of_32_bits(pt, gt, lo):
    P, G = tensors(SIZES, pt, 1, 0.02, lo), tensors(SIZES, gt, 2, 1e-3, lo)
    M, V = tensors(SIZES, torch.float32, 3, 1e-3, lo), [t.square() for t in tensors(SIZES, torch.float32, 4, 1e-3)]
    C = tensors(SIZES, torch.bfloat16, 5, 1.0, lo)
    C[2] = None
    scale = torch.tensor([0.5], device="cuda")
    want = [plain(p, g, m, v, 7, scale=0.5, **HYPER) for p, g, m, v in zip(P, G, M, V)]
    tilec.ext.adamw_step(P, G, M, V, step=7, grad_scale=scale, copies=C, **HYPER)
    for p, m, v, c, ((rp, rm, rv), (ep, em, ev)) in zip(P, M, V, C, want):
        near(p, rp, ep, 2.0 ** -8 if pt == torch.bfloat16 else 0.0)
        near(m, rm, em)
        near(v, rv, ev)
        if c is not None:
            near(c, rp, ep, 2.0 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize("gt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lo", [0, 3])
def test_states_of_8_bits(gt, lo):
    sizes = SIZES
    P, G = tensors(sizes, torch.float32, 1, 0.02, lo), tensors(sizes, gt, 2, 1e-3, lo)
    g = torch.Generator().manual_seed(6)
    blocks = [-(-n // 256) for n in sizes]
    M, V = [], []
    mc = torch.randint(-127, 128, (sum(sizes) + 7 * len(sizes) + lo,), generator=g).to(torch.int8).cuda()
    vc = torch.randint(0, 256, (sum(sizes) + 7 * len(sizes) + lo,), generator=g).to(torch.uint8).cuda()
    at = lo
    for n, b in zip(sizes, blocks):
        M.append((mc[at:at + n], (torch.rand(b, generator=g) * 1e-3).cuda()))
        V.append((vc[at:at + n], (torch.rand(b, generator=g) * 1e-6).cuda()))
        at += n + 7
    m0, v0 = tilec.ext.adamw_values(M), tilec.ext.adamw_values(V)
    for (c, s), m in zip(M, m0):
        t = c.double() / 127
        near(m, t * t.abs() * s.double().repeat_interleave(256)[:c.numel()], 0.0, 6 * E32)
    for (c, s), v in zip(V, v0):
        near(v, (c.double() / 255) ** 4 * s.double().repeat_interleave(256)[:c.numel()], 0.0, 12 * E32)
    want = [plain(p, g, m, v, 3, **HYPER) for p, g, m, v in zip(P, G, m0, v0)]
    tilec.ext.adamw_step(P, G, M, V, step=3, **HYPER)
    for p, (c, s), (d, r), ((rp, rm, rv), (ep, em, ev)) in zip(P, M, V, want):
        near(p, rp, ep)
        n = p.numel()
        pad = -n % 256
        top = torch.nn.functional.pad(rm.abs(), (0, pad)).view(-1, 256).amax(dim=1)
        etop = torch.nn.functional.pad(em, (0, pad)).view(-1, 256).amax(dim=1)
        near(s, top, etop)
        exact = rm.sign() * 127 * (rm.abs() / top.repeat_interleave(256)[:n]).sqrt()
        # The error of m moves its root: by em / (2 sqrt(m top)), or sqrt(em / top) near 0.
        moved = 127 * (em / top.repeat_interleave(256)[:n]).sqrt()
        assert ((c.double() - exact).abs() <= 0.5 + 1e-4 + moved).all()
        top = torch.nn.functional.pad(rv, (0, pad)).view(-1, 256).amax(dim=1)
        near(r, top, 0.0, 8 * E32)
        exact = 255 * (rv / top.repeat_interleave(256)[:n]) ** 0.25
        assert ((d.double() - exact).abs() <= 0.5 + 1e-4).logical_or((d == 1) & (exact < 1)).all()
        assert ((d > 0) | (rv == 0)).all()


@pytest.mark.gpu
def test_many_tensors_none_grads_and_zero_sizes():
    sizes = [5, 0, 300] * 60  # more than one launch
    P, G = tensors(sizes, torch.float32, 1, 0.1), tensors(sizes, torch.float32, 2, 1e-2)
    states = [tilec.ext.adamw_state(p) for p in P]
    M, V = [s[0] for s in states], [s[1] for s in states]
    G[4] = G[5] = None
    before = [p.clone() for p in P]
    want = [None if g is None else plain(p, g, m, v, 1, **HYPER) for p, g, m, v in zip(P, G, M, V)]
    tilec.ext.adamw_step(P, G, M, V, step=1, **HYPER)
    for p, m, v, old, w in zip(P, M, V, before, want):
        if w is None:
            assert torch.equal(p, old) and not m.any() and not v.any()
            continue
        near(p, w[0][0], w[1][0])
        near(m, w[0][1], w[1][1])
        near(v, w[0][2], w[1][2])
    tilec.ext.adamw_step([], [], [], [], step=1)
    tilec.ext.adamw_step(P[:2], [None, None], M[:2], V[:2], step=1)


@pytest.mark.gpu
def test_zero_states_and_zero_gradients():
    for bits in (32, 8):
        p = torch.ones(600, device="cuda")
        m, v = tilec.ext.adamw_state(p, bits)
        # Nothing has been seen: only the decay moves p, and eps = 0 is 0 / 0.
        tilec.ext.adamw_step([p], [torch.zeros_like(p)], [m], [v], step=1, lr=0.1, weight_decay=0.5)
        assert torch.equal(p, torch.full_like(p, torch.tensor(1 - 0.1 * 0.5).item()))
        g = torch.zeros_like(p)
        g[300] = 2.0
        tilec.ext.adamw_step([p], [g], [m], [v], step=1, lr=0.1, weight_decay=0.0)
        assert abs(p[300].item() - (0.95 - 0.1)) < 1e-6 and p[301].item() == p[0].item()


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_non_finite_gradients_show(value):
    # 32 bits: the value's own parameter; 8 bits: the states of its block.
    p = torch.ones(1024, device="cuda")
    g = torch.full_like(p, 1e-3)
    g[700] = value
    q, (m, v), (m8, v8) = p.clone(), tilec.ext.adamw_state(p), tilec.ext.adamw_state(p, 8)
    tilec.ext.adamw_step([p], [g], [m], [v], step=1)
    tilec.ext.adamw_step([q], [g], [m8], [v8], step=1)
    assert torch.equal(p.isnan(), q.isnan()) and p.isnan().sum() == 1 and p[700].isnan()
    tilec.ext.adamw_step([q], [torch.zeros_like(g)], [m8], [v8], step=2)
    bad = q.isnan()
    assert bad[512:768].all() and not bad[:512].any() and not bad[768:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(bits):
    # One tensor of more than 2^31 values, checked at both ends and around 2^31.
    n = (1 << 31) + 1003
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v = tilec.ext.adamw_state(p, bits)
    near_ends = [slice(0, 512), slice((1 << 31) - 256, (1 << 31) + 256), slice(n - 1003 % 256, n)]
    gen = torch.Generator().manual_seed(7)
    for s in near_ends:
        size = p[s].numel()
        p[s] = torch.randn(size, generator=gen).cuda()
        g[s] = (torch.randn(size, generator=gen) * 1e-3).cuda()
    want = [plain(p[s], g[s], torch.zeros_like(p[s]), torch.zeros_like(p[s]), 1, **HYPER) for s in near_ends]
    tilec.ext.adamw_step([p], [g], [m], [v], step=1, **HYPER)
    for s, ((rp, rm, rv), (ep, em, ev)) in zip(near_ends, want):
        near(p[s], rp, ep, 2.0 ** -8)
        if bits == 32:
            near(m[s], rm, em)
            near(v[s], rv, ev)
        else:
            assert (m[0][s].sign() == rm.sign()).logical_or(m[0][s] == 0).all() and (v[0][s] > 0).all()
    assert not p[1 << 20:1 << 21].any()


@pytest.mark.gpu
def test_8_bits_train_like_32():
    # A least-squares problem of 64 x 512 unknowns with noisy gradients.
    g = torch.Generator().manual_seed(3)
    goal = torch.randn(64, 512, generator=g).cuda()
    scale = torch.logspace(-2, 0, 512).cuda()  # curvatures over two orders
    noise = torch.randn(100, 64, 512, generator=g).cuda()
    left = {}
    for bits in (32, 8):
        p = torch.zeros(64, 512, device="cuda")
        m, v = tilec.ext.adamw_state(p, bits)
        for step in range(1, 301):
            grad = (p - goal) * scale + 0.1 * scale * noise[step % 100]
            tilec.ext.adamw_step([p], [grad], [m], [v], step=step, lr=2e-2, weight_decay=0.0)
        left[bits] = ((p - goal).square().mean() / goal.square().mean()).item()
    assert left[32] < 0.02 and left[8] < 1.5 * left[32] + 0.01


@pytest.mark.gpu
def test_another_stream():
    sizes = [100, 5000, 40000]
    runs = []
    for stream in (None, torch.cuda.Stream()):
        P, G = tensors(sizes, torch.float32, 1, 0.02), tensors(sizes, torch.bfloat16, 2, 1e-3)
        states = [tilec.ext.adamw_state(p, 8) for p in P]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            tilec.ext.adamw_step(P, G, [s[0] for s in states], [s[1] for s in states], step=1)
        torch.cuda.synchronize()
        runs.append(P + [s[0][0] for s in states] + [s[1][1] for s in states])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
def test_refusals():
    f = tilec.ext.adamw_step
    p, g = torch.zeros(6, 4, device="cuda"), torch.zeros(6, 4, device="cuda")
    m, v = tilec.ext.adamw_state(p)
    m8, v8 = tilec.ext.adamw_state(p, 8)
    ok = {"step": 1}
    for args, kw, error in (
            (([p], [g, g], [m], [v]), ok, ValueError), (([p], [g[:5]], [m], [v]), ok, ValueError),
            (([p], [g], [m[:5]], [v]), ok, ValueError), (([p], [g], [m], [v]), {"step": 0}, ValueError),
            (([p], [g], [m], [v]), {"step": 1, "betas": (1.0, 0.9)}, ValueError),
            (([p], [g], [m], [v]), {"step": 1, "lr": -1.0}, ValueError),
            (([p], [g], [m], [v]), {"step": 1, "eps": float("nan")}, ValueError),
            (([p.t()], [g], [m], [v]), ok, ValueError), (([p, p], [g, g], [m, m], [v, v]), ok, ValueError),
            (([p.half()], [g], [m], [v]), ok, TypeError), (([p], [g.half()], [m], [v]), ok, TypeError),
            (([p], [g], [m.bfloat16()], [v]), ok, TypeError), (([p], [g], [m8], [v]), ok, ValueError),
            (([p], [g], [m8], [m8]), ok, TypeError), (([p], [g], [(m8[0], m8[1][:0])], [v8]), ok, ValueError),
            (([p], [g.cpu()], [m], [v]), ok, TypeError), (([p.cpu()], [g], [m], [v]), ok, TypeError),
            (([p], [g], [m], [v]), {"step": 1, "copies": [p]}, TypeError),
            (([p], [g], [m], [v]), {"step": 1, "copies": []}, ValueError),
            (([p], [g], [m], [v]), {"step": 1, "grad_scale": torch.ones(2, device="cuda")}, ValueError),
            (([p], [g], [m], [v]), {"step": 1, "grad_scale": torch.ones(1)}, TypeError)):
        with pytest.raises(error):
            f(*args, **kw)
    assert not p.any() and not m.any() and not v.any()
    with pytest.raises(ValueError):
        tilec.ext.adamw_state(p, 16)
    with pytest.raises(ValueError):
        tilec.ext.adamw_values([m])
    with pytest.raises(TypeError):
        tilec.ext.adamw_values([(m, m8[1])])


def test_cpu_tensors_are_refused():
    p = torch.zeros(3)
    m, v = tilec.ext.adamw_state(p)
    with pytest.raises(TypeError):
        tilec.ext.adamw_step([p], [p], [m], [v], step=1)
    with pytest.raises(TypeError):
        tilec.ext.adamw_values([tilec.ext.adamw_state(p, 8)[0]])
