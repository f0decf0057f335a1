"""Cross entropy of a linear layer's outputs and its gradients against plain
64-bit forms, at the sizes, types, masks and values where they can go wrong.

Tolerances.  A logit is a sum of H products in fp32: its error is at most
(H + 2) 2^-24 of the sum of their magnitudes, `elogit` below, and the loss's
at most twice that of the row's largest, plus the roundings of exp, the sums
of exp and log (their chains are under 300 additions: 300 2^-24, and 4
roundings of the loss), `erow`.  softmax has twice that as its relative error,
and so has d = g (softmax - onehot), but at the target, where it is 2 erow g;
for bf16 inputs d is rounded to fp16 before and to bf16 after it is scaled,
2^-11 + 2^-8, and what is below 2^-39 of a group's largest exp is dropped or
kept to that.  The gradients add the error of their own sums, (their length +
2) 2^-24, and one rounding of the result.
"""

import math

import pytest
import torch

import tilec

E32 = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(N, H, V, dt, seed=0, ignored=0.0, std=2.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, H, generator=g) * (std / math.sqrt(H))
    t = torch.randint(V, (N,), generator=g)
    x = torch.randn(N, H, generator=g) + 0.7 * w[t]
    if ignored:
        t[torch.rand(N, generator=g) < ignored] = -100
    return x.to(TYPES[dt]).cuda(), w.to(TYPES[dt]).cuda(), t.cuda()


def plain(x, w, t, reduction="mean", grad_loss=None, ignore=-100):
    """(loss, dx, dw, d, g): 64-bit values, the gradient of the logits and its
    rows' factors."""
    x, w = x.double(), w.double()
    N = x.shape[0]
    keep = t != ignore
    logits = x @ w.t().contiguous()
    at = torch.where(keep, t, 0)[:, None]
    lse = logits.logsumexp(dim=1)
    rows = torch.where(keep, lse - logits.gather(1, at)[:, 0], 0.0)
    d = (logits - lse[:, None]).exp().scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    g = torch.ones(N, dtype=torch.float64, device=x.device)
    if grad_loss is not None:
        g = g * grad_loss.double()
    count = max(1, int(keep.sum()))
    if reduction == "mean":
        g = g / count
    g = g * keep
    d = d * g[:, None]
    loss = rows if reduction == "none" else rows.sum() / (count if reduction == "mean" else 1)
    return loss, d @ w, d.t().contiguous() @ x, d, g.abs()


def bounds(x, w, t, d, g):
    """Error bounds of the per-row losses, of dx and of dw."""
    xa, wa = x.double().abs(), w.double().abs()
    N, H = x.shape
    V = w.shape[0]
    erow = 2 * (H + 2) * E32 * (xa @ wa.t().contiguous()).amax(dim=1) + 300 * E32
    bf16 = x.dtype == torch.bfloat16
    ed = d.abs() * (2 * erow + (2.0 ** -8 + 2.0 ** -11 if bf16 else 4 * E32))[:, None]
    if bf16:
        ed = ed + 2.0 ** -38 * g[:, None]
    rows = torch.arange(N, device=t.device)
    ed[rows, torch.where((t >= 0) & (t < V), t, 0)] += 2 * erow * g
    edx = ed @ wa + (V + 2) * E32 * (d.abs() @ wa)
    edw = ed.t().contiguous() @ xa + (N + 2) * E32 * (d.abs().t().contiguous() @ xa)
    return erow, edx, edw


def check(x, w, t, reduction="mean", grad_loss=None, chunk_rows=0, ignore=-100):
    loss, dx, dw = tilec.ext.linear_cross_entropy_grad(x, w, t, reduction, ignore, grad_loss, chunk_rows)
    only = tilec.ext.linear_cross_entropy(x, w, t, reduction, ignore)
    rl, rdx, rdw, d, g = plain(x, w, t, reduction, grad_loss, ignore)
    erow, edx, edw = bounds(x, w, t, d, g)
    erow = torch.where(t == ignore, 0.0, erow)
    if reduction == "none":
        el = erow + 4 * E32 * rl.abs()
    else:
        n = max(1, int((t != ignore).sum())) if reduction == "mean" else 1
        el = erow.sum() / n + 4 * E32 * rl.abs()
    out = 2.0 ** -8 if x.dtype == torch.bfloat16 else E32
    assert loss.dtype == torch.float32 and dx.dtype == dw.dtype == x.dtype
    assert loss.shape == rl.shape and dx.shape == x.shape and dw.shape == w.shape
    assert ((loss.double() - rl).abs() <= el).all()
    assert ((only.double() - rl).abs() <= el).all()
    assert ((dx.double() - rdx).abs() <= edx + out * (rdx.abs() + edx) + 1e-37).all()
    assert ((dw.double() - rdw).abs() <= edw + out * (rdw.abs() + edw) + 1e-37).all()
    return loss, dx, dw


SHAPES = [(1, 8, 2), (1, 64, 1), (3, 5, 7), (7, 1024, 1000), (64, 64, 64), (65, 72, 129), (130, 100, 1003),
          (257, 192, 5003), (1000, 333, 777), (300, 640, 8200), (16, 1, 40), (2, 4096, 30011)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("N,H,V", SHAPES)
def test_loss_and_gradients(N, H, V, dt):
    x, w, t = make(N, H, V, dt, seed=N + H + V, ignored=0.25 if N > 3 else 0.0)
    got = check(x, w, t)
    again = tilec.ext.linear_cross_entropy_grad(x, w, t)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # the same bits
    g = torch.Generator().manual_seed(1)
    check(x, w, t, "none", torch.randn(N, generator=g).cuda())
    check(x, w, t, "sum", torch.tensor(-0.37, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("N,H,V,rows", [(300, 128, 1001, 128), (300, 130, 1000, 100), (257, 64, 300, 256), (5, 24, 33, 1)])
def test_chunks(N, H, V, rows, dt):
    x, w, t = make(N, H, V, dt, seed=3, ignored=0.2)
    check(x, w, t, chunk_rows=rows)
    check(x, w, t, "none", chunk_rows=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("N,H,V,rows", [(2304, 2304, 16500, 0), (600, 520, 25000, 0), (600, 520, 25000, 512),
                                        (1300, 130, 40000, 0)])
def test_many_tiles(N, H, V, rows):
    # Enough output tiles for the largest ones, in whole turns over the chip and
    # with a rest in smaller ones.
    x, w, t = make(N, H, V, "bf16", seed=4, ignored=0.1)
    check(x, w, t, chunk_rows=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("N,H,V", [(640, 928, 978), (100, 520, 3000), (40, 200, 1000), (9, 72, 257), (2048, 1000, 16000)])
def test_widths_of_no_whole_steps(N, H, V, dt):
    # Whatever lies past a row's end must not get in.
    x, w, t = make(N, H, V, dt, seed=H, ignored=0.1)
    wide_x = torch.full((N + 1, H + 8), math.nan, dtype=x.dtype, device="cuda")
    wide_w = torch.full((V + 1, H + 16), math.nan, dtype=x.dtype, device="cuda")
    wide_x[:N, :H], wide_w[:V, :H] = x, w
    got = check(wide_x[:N, :H], wide_w[:V, :H], t)
    assert all(torch.equal(a, b) for a, b in zip(got, tilec.ext.linear_cross_entropy_grad(x, w, t)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("N,H,V", [(2047, 64, 130), (2050, 40, 1), (4099, 72, 1001), (6001, 16, 4097), (2049, 64, 16500)])
def test_many_rows(N, H, V, dt):
    # About where rows are given a wave or a workgroup each, by their number and
    # length.
    x, w, t = make(N, H, V, dt, seed=N + V, ignored=0.2)
    t[N - 1] = V - 1
    check(x, w, t)
    g = torch.Generator().manual_seed(2)
    check(x, w, t, "none", torch.randn(N, generator=g).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 40])
def test_offsets_past_32_bits(N):
    # A weight and a gradient of more than 2^31 values, checked for the last
    # classes and the targets'.  x is zero but in 64 columns, the last one among
    # them: what the logits and dw round is the sums of those alone, so that the
    # bounds stay as narrow as those of a small problem.
    H, V, L = 32776, 65600, 64
    g = torch.Generator(device="cuda").manual_seed(12)
    w = torch.randn(V, H, generator=g, device="cuda", dtype=torch.bfloat16).mul_(0.25)
    cols = torch.cat([torch.randperm(H - 1, generator=g, device="cuda")[:L - 1], torch.tensor([H - 1], device="cuda")])
    x = torch.zeros(N, H, device="cuda", dtype=torch.bfloat16)
    x[:, cols] = torch.randn(N, L, generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randint(V, (N,), generator=g, device="cuda")
    t[0] = V - 1
    loss, dx, dw = tilec.ext.linear_cross_entropy_grad(x, w, t, "sum")
    xl, wl = x[:, cols], w[:, cols]
    rl, _, rdw, d, gr = plain(xl, wl, t, "sum")
    erow, _, edw = bounds(xl, wl, t, d, gr)
    assert (loss.double() - rl).abs() <= erow.sum() + 4 * E32 * rl.abs()
    assert ((dw[:, cols].double() - rdw).abs() <= edw + 2.0 ** -8 * (rdw.abs() + edw)).all()
    rest = torch.ones(H, dtype=torch.bool, device="cuda")
    rest[cols] = False
    assert not dw[-300:, rest].any() and not dw[t][:, rest].any()
    # dx for a few columns of w, the last one among them.
    some = torch.cat([torch.arange(8, device="cuda"), torch.arange(H - 56, H, device="cuda")])
    ws = w[:, some].double()
    ed = d.abs() * (2 * erow + 2.0 ** -8 + 2.0 ** -11)[:, None] + 2.0 ** -38
    ed[torch.arange(N, device="cuda"), t] += 2 * erow
    edx = ed @ ws.abs() + (V + 2) * E32 * (d.abs() @ ws.abs())
    rdx = d @ ws
    assert ((dx[:, some].double() - rdx).abs() <= edx + 2.0 ** -8 * (rdx.abs() + edx)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_views(dt):
    # Rows of wider matrices, aligned and from an odd element on.
    g = torch.Generator().manual_seed(2)
    for lo in (0, 3):
        xs = torch.randn(70, 200, generator=g).to(TYPES[dt]).cuda()
        ws = torch.randn(500, 264, generator=g).mul_(0.2).to(TYPES[dt]).cuda()
        t = torch.randint(500, (140,), generator=g).cuda()[::2]
        check(xs[:, lo:lo + 136], ws[:, lo:lo + 136], t)
    # Transposed: copied.
    check(xs.t()[:136].contiguous().t()[:, :136], ws.t()[:136].t(), t)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_ignored_rows(dt):
    x, w, t = make(200, 64, 301, dt, seed=6, ignored=0.4)
    want = check(x, w, t)
    # What an ignored row holds reaches nothing.
    bad = x.clone()
    rows = (t == -100).nonzero()[:, 0]
    bad[rows[0]], bad[rows[1]], bad[rows[2], 5] = float("nan"), float("inf"), float("-inf")
    got = tilec.ext.linear_cross_entropy_grad(bad, w, t)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert not got[1][rows].any()
    assert torch.equal(tilec.ext.linear_cross_entropy(bad, w, t, "none"), tilec.ext.linear_cross_entropy(x, w, t, "none"))
    # Another ignore_index, a class of its own.
    check(x, w, torch.where(t == -100, 7, t), ignore=7)
    # No row that counts: 0, and gradients of zeros.
    none = torch.full_like(t, -100)
    for reduction in ("mean", "sum", "none"):
        loss, dx, dw = tilec.ext.linear_cross_entropy_grad(bad, w, none, reduction)
        assert not loss.any() and not dx.any() and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_no_rows(dt):
    x, w, t = make(0, 16, 9, dt)
    loss, dx, dw = tilec.ext.linear_cross_entropy_grad(x, w, t)
    assert loss.item() == 0 and dx.shape == (0, 16) and not dw.any() and dw.shape == (9, 16)
    assert tilec.ext.linear_cross_entropy(x, w, t, "none").shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_large_and_infinite_logits(dt):
    # Logits in the hundreds: nothing overflows, one class takes all.
    x, w, t = make(40, 64, 500, dt, seed=8, std=60.0)
    check(x, w, t)
    # A class whose logits are all -inf (a weight row of -inf against positive
    # features) takes no part, as a vocabulary entry masked out; as a target it
    # costs an infinite loss.
    x = x.abs() + 0.1
    w = (w / 60).clone()
    w[11] = float("-inf")
    t = torch.where(t == 11, 12, t)
    want = tilec.ext.linear_cross_entropy(x, torch.cat([w[:11], w[12:]]), torch.where(t > 11, t - 1, t), "none")
    got = tilec.ext.linear_cross_entropy(x, w, t, "none")
    assert ((got - want).abs() <= 1e-5 * (1 + want.abs())).all()
    t[0] = 11
    assert tilec.ext.linear_cross_entropy(x, w, t, "none")[0].item() == math.inf
    # A NaN stays in its row's loss.
    x, w, t = make(40, 64, 500, dt, seed=8)
    x[5, 3] = float("nan")
    loss = tilec.ext.linear_cross_entropy(x, w, t, "none")
    assert loss[5].isnan() and not loss[[i for i in range(40) if i != 5]].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_target_that_is_no_class(dt):
    x, w, t = make(30, 64, 100, dt, seed=9)
    good = tilec.ext.linear_cross_entropy(x, w, t, "none")
    for value in (100, -1, 1 << 40, -(1 << 40)):
        bad = t.clone()
        bad[4] = value
        loss = tilec.ext.linear_cross_entropy(x, w, bad, "none")
        assert loss[4].isnan() and torch.equal(loss[5:], good[5:])
        loss, dx, dw = tilec.ext.linear_cross_entropy_grad(x, w, bad)
        assert loss.isnan() and dx[4].isnan().all() and dw.isnan().all()


@pytest.mark.gpu
def test_gradients_against_differences():
    # Central differences of the 64-bit loss; h^2 times its third derivative
    # and 2^-52 / h are both under 1e-8.
    x, w, t = make(3, 6, 5, "f32", seed=10)
    loss, dx, dw = (v.cpu().double() for v in tilec.ext.linear_cross_entropy_grad(x, w, t))
    x, w, t = x.cpu().double(), w.cpu().double(), t.cpu()
    h = 1e-4
    for v, grad in ((x, dx), (w, dw)):
        flat, got = v.view(-1), grad.reshape(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + h
            up = plain(x, w, t)[0]
            flat[i] = keep - h
            down = plain(x, w, t)[0]
            flat[i] = keep
            assert abs((up - down) / (2 * h) - got[i]) <= 3e-6


@pytest.mark.gpu
def test_another_stream():
    x, w, t = make(256, 512, 4000, "bf16", seed=11, ignored=0.1)
    want = tilec.ext.linear_cross_entropy_grad(x, w, t)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = tilec.ext.linear_cross_entropy_grad(x, w, t)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_refusals():
    f, g = tilec.ext.linear_cross_entropy, tilec.ext.linear_cross_entropy_grad
    x, w, t = make(4, 8, 10, "f32")
    for bad, error in (((x[0], w, t), ValueError), ((x, w[:, :7], t), ValueError), ((x, w, t[:3]), ValueError),
                       ((x, w, t, "median"), ValueError), ((x, w.bfloat16(), t), TypeError),
                       ((x.half(), w.half(), t), TypeError), ((x, w, t.int()), TypeError),
                       ((x, w.cpu(), t), TypeError), ((x, w, t.cpu()), TypeError),
                       ((x[:, :0], w[:, :0], t), ValueError), ((x, w[:0], t), ValueError)):
        with pytest.raises(error):
            f(*bad)
        with pytest.raises(error):
            g(*bad)
    for kw, error in (({"grad_loss": torch.ones(4, device="cuda")}, ValueError),
                      ({"grad_loss": torch.ones((), device="cuda", dtype=torch.float64)}, TypeError),
                      ({"grad_loss": torch.ones(())}, TypeError), ({"chunk_rows": -1}, ValueError)):
        with pytest.raises(error):
            g(x, w, t, **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(TypeError):
        tilec.ext.linear_cross_entropy(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64))
