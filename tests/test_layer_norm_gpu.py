"""Layer norm and its gradients against plain 64-bit forms, at the sizes, types,
strides and values where they can go wrong.

Tolerances.  A sum of n terms is added in a chain of at most 64 additions a
thread, 10 steps across threads and, for column sums, R / parts rows a thread
and parts more: its error is below (chain length) 2^-24 of the sum of the
terms' magnitudes, and every term carries a few roundings of its own.  bf16
outputs add one rounding, 2^-8 of the value (2^-9 of its binade's top).
"""

import pytest
import torch

import tilec

E32 = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 64), (17, 257), (300, 1009), (4099, 16), (33, 4096), (9, 16384), (7, 16385),
          (3, 20000), (2, 70001), (600, 129), (2500, 512)]


def make(R, D, xt, yt, wt, seed=0, offset=0.25):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, D, generator=g) * 1.5 + offset).to(TYPES[xt]).cuda()
    w = (torch.randn(D, generator=g) * 0.2 + 1).to(TYPES[wt]).cuda()
    b = (torch.randn(D, generator=g) * 0.1).to(TYPES[wt]).cuda()
    dy = torch.randn(R, D, generator=g).to(TYPES[yt]).cuda()
    return x, w, b, dy


def plain(x, w, b, eps=1e-5):
    x = x.double()
    mean = x.mean(dim=1)
    dev = x - mean[:, None]
    rstd = (dev.square().mean(dim=1) + eps) ** -0.5
    y = dev * rstd[:, None]
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd


def plain_grad(dy, x, mean, rstd, w):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    xhat = (x - mean) * rstd
    wdy = dy if w is None else dy * w.double()
    c1, c2 = wdy.mean(dim=1, keepdim=True), (wdy * xhat).mean(dim=1, keepdim=True)
    return rstd * (wdy - c1 - xhat * c2), (dy * xhat).sum(dim=0), dy.sum(dim=0)


def half_ulp(t):
    return 2.0 ** -8 if t == torch.bfloat16 else E32


def check_forward(x, w, b, y, mean, rstd, eps=1e-5):
    ry, rmean, rrstd = plain(x, w, b, eps)
    # The mean's error is at most 80 roundings of the mean magnitude; it moves
    # the deviations, and by them xhat.
    mag = x.double().abs().mean(dim=1)
    emean = 80 * E32 * mag
    assert ((mean.double() - rmean).abs() <= emean + 1e-37).all()
    erstd = rrstd * (90 * E32 + emean * rrstd)
    assert ((rstd.double() - rrstd).abs() <= erstd).all()
    wmag = 1.0 if w is None else w.double().abs()
    xhat = (x.double() - rmean[:, None]).abs() * rrstd[:, None]
    tol = wmag * (emean * rrstd)[:, None] + wmag * xhat * (100 * E32 + (emean * rrstd)[:, None]) + 4 * E32
    tol = tol + ry.abs() * (half_ulp(y.dtype) + 4 * E32)
    assert ((y.double() - ry).abs() <= tol).all()


def check_backward(dy, x, mean, rstd, w, dx, dw, db):
    rdx, rdw, rdb = plain_grad(dy, x, mean, rstd, w)
    R, D = x.shape
    xhat = ((x.double() - mean.double()[:, None]) * rstd.double()[:, None]).abs()
    wdy = dy.double().abs() if w is None else (dy.double() * w.double()).abs()
    # xhat itself: x - mean rounds to 2^-24 of its larger operand.
    exhat = E32 * (2 * xhat + rstd.double()[:, None] * mean.double().abs()[:, None])
    c1, c2 = wdy.mean(dim=1, keepdim=True), (wdy * xhat).mean(dim=1, keepdim=True)
    ec = 90 * E32
    tol = rstd.double()[:, None] * (wdy * 4 * E32 + c1 * ec + xhat * c2 * ec + exhat * c2
                                    + xhat * (wdy * exhat).mean(dim=1, keepdim=True))
    assert ((dx.double() - rdx).abs() <= tol + rdx.abs() * (half_ulp(dx.dtype) + 4 * E32) + 1e-37).all()
    chain = (R + 64) * E32
    adw = (dy.double().abs() * xhat).sum(dim=0)
    assert ((dw.double() - rdw).abs() <= chain * adw + (dy.double().abs() * exhat).sum(dim=0) + 1e-37).all()
    assert ((db.double() - rdb).abs() <= chain * dy.double().abs().sum(dim=0) + 1e-37).all()


@pytest.mark.gpu
@pytest.mark.parametrize("xt,yt,wt", [("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "bf16"),
                                      ("bf16", "f32", "f32")])
@pytest.mark.parametrize("R,D", SHAPES)
def test_both_passes(R, D, xt, yt, wt):
    x, w, b, dy = make(R, D, xt, yt, wt, seed=R + D)
    y, mean, rstd = tilec.ext.layer_norm(x, w, b, dtype=TYPES[yt])
    assert y.dtype == TYPES[yt] and y.shape == x.shape and mean.dtype == rstd.dtype == torch.float32
    check_forward(x, w, b, y, mean, rstd)
    dx, dw, db = tilec.ext.layer_norm_backward(dy, x, mean, rstd, w)
    assert dx.dtype == dy.dtype and dw.dtype == db.dtype == torch.float32
    check_backward(dy, x, mean, rstd, w, dx, dw, db)
    again = tilec.ext.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))  # the same bits
    only = tilec.ext.layer_norm_backward(dy, x, mean, rstd, w, param_grads=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_views_and_missing_parameters(dt):
    # Rows of a wider matrix from an odd element on; parameters at odd elements.
    x, w, b, dy = make(70, 333, dt, dt, dt)
    xv, dyv = x[:, 5:300], dy[:, 3:298]
    wv, bv = w[1:296], b[3:298]
    y, mean, rstd = tilec.ext.layer_norm(xv, wv, bv)
    check_forward(xv, wv, bv, y, mean, rstd)
    check_backward(dyv, xv, mean, rstd, wv, *tilec.ext.layer_norm_backward(dyv, xv, mean, rstd, wv))
    # Columns of a transposed matrix: copied.
    xt = x.t()[:256]
    y, mean, rstd = tilec.ext.layer_norm(xt)
    check_forward(xt, None, None, y, mean, rstd)
    dyt = dy.t()[:256]
    check_backward(dyt, xt, mean, rstd, None, *tilec.ext.layer_norm_backward(dyt, xt, mean, rstd))
    y, mean, rstd = tilec.ext.layer_norm(xv, None, bv)
    check_forward(xv, None, bv, y, mean, rstd)
    # One row, one dimension.
    y, mean, rstd = tilec.ext.layer_norm(x[4], w, b)
    assert y.shape == (333,) and mean.shape == (1,)
    check_forward(x[4:5], w, b, y[None], mean, rstd)
    # A broadcast row: stride 0.
    xb = x[:1].expand(6, 333)
    y, mean, rstd = tilec.ext.layer_norm(xb, w, b)
    check_forward(xb, w, b, y, mean, rstd)


@pytest.mark.gpu
def test_wide_row_stride():
    # Rows whose offsets pass 32 bits (in bytes).
    store = torch.empty((3, 1 << 29), dtype=torch.float32, device="cuda")
    x, w, b, dy = make(3, 1000, "f32", "f32", "f32")
    store[:, :1000] = x
    v = store[:, :1000]
    y, mean, rstd = tilec.ext.layer_norm(v, w, b)
    check_forward(x, w, b, y, mean, rstd)
    check_backward(dy, x, mean, rstd, w, *tilec.ext.layer_norm_backward(dy, v, mean, rstd, w))


@pytest.mark.gpu
def test_constant_rows_large_means_and_special_values():
    x = torch.full((4, 100), 3.0, device="cuda")
    y, mean, rstd = tilec.ext.layer_norm(x)
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(mean, x[:, 0])
    # A mean a thousand times the deviation: the variance comes from deviations.
    x, w, b, dy = make(50, 777, "f32", "f32", "f32", offset=1500.0)
    check_forward(x, w, b, *tilec.ext.layer_norm(x, w, b))
    # A row with an infinity or a NaN spoils that row and no other.
    x, w, b, dy = make(9, 300, "f32", "f32", "f32")
    good = tilec.ext.layer_norm(x, w, b)
    x[3, 17], x[5, 299] = float("inf"), float("nan")
    y, mean, rstd = tilec.ext.layer_norm(x, w, b)
    keep = [0, 1, 2, 4, 6, 7, 8]
    assert torch.equal(y[keep], good[0][keep])
    assert y[3].isnan().all() and y[5].isnan().all()


@pytest.mark.gpu
def test_no_rows():
    x = torch.empty((0, 40), device="cuda")
    y, mean, rstd = tilec.ext.layer_norm(x)
    assert y.shape == (0, 40) and mean.shape == (0,)
    dx, dw, db = tilec.ext.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 40) and torch.equal(dw, torch.zeros(40, device="cuda")) and torch.equal(db, dw)


@pytest.mark.gpu
def test_gradients_against_differences():
    # Central differences of sum(dy * y) in 64 bits; their own error is
    # h^2 times a third derivative, about 1e-8 here, and 2^-52 / h.
    x, w, b, dy = make(2, 13, "f32", "f32", "f32", seed=5)
    y, mean, rstd = tilec.ext.layer_norm(x, w, b)
    dx, dw, db = (t.cpu().double() for t in tilec.ext.layer_norm_backward(dy, x, mean, rstd, w))
    x, w, b, dy = (t.cpu().double() for t in (x, w, b, dy))

    def f():
        return (dy * plain(x, w, b)[0]).sum()

    h = 1e-4
    for t, grad in ((x, dx), (w, dw), (b, db)):
        flat, got = t.view(-1), grad.reshape(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + h
            up = f()
            flat[i] = keep - h
            down = f()
            flat[i] = keep
            assert abs((up - down) / (2 * h) - got[i]) <= 3e-6 * (1 + abs(got[i]))


@pytest.mark.gpu
def test_another_stream():
    x, w, b, dy = make(512, 1024, "bf16", "bf16", "bf16")
    want = tilec.ext.layer_norm(x, w, b)
    grads = tilec.ext.layer_norm_backward(dy, x, want[1], want[2], w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = tilec.ext.layer_norm(x, w, b)
        got_grads = tilec.ext.layer_norm_backward(dy, x, got[1], got[2], w)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want + grads, got + got_grads))


@pytest.mark.gpu
def test_refusals():
    f, g = tilec.ext.layer_norm, tilec.ext.layer_norm_backward
    x, w, b, dy = make(4, 8, "f32", "f32", "f32")
    stat = torch.zeros(4, device="cuda")
    for bad, error in (((x[None],), ValueError), ((x, w[:7]), ValueError), ((x, w, b.bfloat16()), TypeError),
                       ((x.half(),), TypeError), ((x, w.half()), TypeError), ((x, w.cpu()), TypeError),
                       ((torch.empty((3, 0), device="cuda"),), ValueError)):
        with pytest.raises(error):
            f(*bad)
    with pytest.raises(TypeError):
        f(x, dtype=torch.float16)
    for bad, error in (((dy[:3], x, stat, stat), ValueError), ((dy, x, stat[:3], stat), ValueError),
                       ((dy, x, stat, stat.double()), TypeError), ((dy.double(), x, stat, stat), TypeError),
                       ((dy, x, stat, stat, w[1:]), ValueError), ((dy, x.cpu(), stat, stat), TypeError)):
        with pytest.raises(error):
            g(*bad)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3)
    with pytest.raises(TypeError):
        tilec.ext.layer_norm(x)
    with pytest.raises(TypeError):
        tilec.ext.layer_norm_backward(x, x, torch.zeros(2), torch.ones(2))
