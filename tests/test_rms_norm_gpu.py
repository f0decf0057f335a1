"""Root mean square norm and its gradients against plain 64-bit forms, at the
sizes, types, strides and values where they can go wrong.

Tolerances.  The sum of D squares is added in a chain of at most 72 additions a
thread and 10 steps across threads, all of one sign: below 90 2^-24 of itself, half
of that in rstd.  Column sums chain R / parts rows a thread and parts more: below R
+ 64 roundings of their terms' magnitudes.  bf16 outputs add one rounding, 2^-8 of
the value.
"""

import pytest
import torch

import tilec

E32 = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
# A value's distance from its code: half a step, 2^-4 or 2^-3 of the value, and
# below the normal range half of the smallest step.
HALF_STEP = {"e4m3": (2.0 ** -4, 2.0 ** -10), "e5m2": (2.0 ** -3, 2.0 ** -17)}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 64), (17, 257), (300, 1009), (4099, 16), (33, 4096), (9, 16384), (7, 16385),
          (3, 20000), (2, 70001), (600, 129), (2500, 512), (5000, 100)]


def make(R, D, xt, rt="", wt="f32", seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, D, generator=g) * 1.5 + 0.25).to(TYPES[xt]).cuda()
    res = (torch.randn(R, D, generator=g) * 2).to(TYPES[rt]).cuda() if rt else None
    w = (torch.randn(D, generator=g) * 0.2 + 1).to(TYPES[wt]).cuda()
    return x, res, w


def half_ulp(t):
    return 2.0 ** -8 if t == torch.bfloat16 else E32


def check_forward(x, res, w, y, h, rstd, eps=1e-5):
    if res is None:
        assert h.data_ptr() == x.data_ptr()
    else:
        assert h.dtype == res.dtype and torch.equal(h, (x.float() + res.float()).to(res.dtype))
    hd = h.double()
    want = (hd.square().mean(dim=1) + eps) ** -0.5
    assert rstd.dtype == torch.float32
    assert ((rstd.double() - want).abs() <= 50 * E32 * want).all()
    ry = hd * want[:, None] * (1 if w is None else w.double())
    if isinstance(y, tuple):
        return check_codes(ry, *y, rel=60 * E32)
    assert y.shape == x.shape
    assert ((y.double() - ry).abs() <= ry.abs() * (60 * E32 + half_ulp(y.dtype))).all()


def check_codes(want, codes, scales, rel):
    """Codes and scales of rows' blocks that stand for `want`, which the kernel had
    to within `rel` of itself."""
    name = {v: k for k, v in TYPES.items()}[codes.dtype]
    R, D = want.shape
    assert codes.shape == want.shape and scales.shape == (R, -(-D // 128)) and scales.dtype == torch.float32
    padded = torch.nn.functional.pad(want, (0, -D % 128)).view(R, -1, 128)
    top = padded.abs().amax(dim=2).clamp(min=2.0 ** -100)
    assert ((scales.double() * LARGEST[name] - top).abs() <= top * (rel + 4 * E32)).all()
    each = scales.double().repeat_interleave(128, dim=1)[:, :D]
    half, low = HALF_STEP[name]
    tol = want.abs() * (half + rel + 4 * E32) + low * each
    assert ((codes.double() * each - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("xt,rt,yt,wt", [("f32", "", "f32", "f32"), ("bf16", "bf16", "bf16", "bf16"),
                                         ("f32", "bf16", "bf16", "bf16"), ("bf16", "f32", "f32", "f32"),
                                         ("bf16", "bf16", "e4m3", "bf16"), ("f32", "f32", "e5m2", "f32"),
                                         ("bf16", "", "e5m2", "f32"), ("f32", "bf16", "e4m3", "f32")])
@pytest.mark.parametrize("R,D", SHAPES)
def test_forward(R, D, xt, rt, yt, wt):
    x, res, w = make(R, D, xt, rt, wt, seed=R + D)
    y, h, rstd = tilec.ext.rms_norm(x, w, res, dtype=TYPES[yt])
    assert (y[0] if isinstance(y, tuple) else y).dtype == TYPES[yt]
    check_forward(x, res, w, y, h, rstd)


@pytest.mark.gpu
@pytest.mark.parametrize("xt,yt", [("bf16", "e4m3"), ("f32", "e5m2")])
@pytest.mark.parametrize("R,D", [(40, 4096), (3, 1000), (2100, 384), (2, 40000)])
def test_codes_are_those_of_the_float32_output(R, D, xt, yt):
    x, res, w = make(R, D, xt, "f32", "f32", seed=3)
    codes, scales = tilec.ext.rms_norm(x, w, res, dtype=TYPES[yt])[0]
    y = tilec.ext.rms_norm(x, w, res, dtype=torch.float32)[0]
    want, ws = tilec.ext.quantize_fp8(y, dtype=TYPES[yt])
    assert torch.equal(scales, ws)
    assert torch.equal(codes.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("ht,yt,dt,wt", [("f32", "f32", "", "f32"), ("bf16", "bf16", "", "bf16"),
                                         ("bf16", "bf16", "bf16", "bf16"), ("f32", "bf16", "f32", "bf16"),
                                         ("bf16", "f32", "bf16", "f32"), ("bf16", "bf16", "f32", "f32"),
                                         ("f32", "f32", "bf16", "f32")])
@pytest.mark.parametrize("R,D", SHAPES)
def test_backward(R, D, ht, yt, dt, wt):
    h, dh, w = make(R, D, ht, dt, wt, seed=R + D)
    dy = torch.randn(R, D, generator=torch.Generator().manual_seed(R)).to(TYPES[yt]).cuda()
    rstd = tilec.ext.rms_norm(h, w)[2]
    dx, dw = tilec.ext.rms_norm_backward(dy, h, rstd, w, dh=dh)
    assert dx.dtype == (dy if dh is None else dh).dtype and dw.dtype == torch.float32
    check_backward(dy, h, rstd, w, dh, dx, dw)
    again = tilec.ext.rms_norm_backward(dy, h, rstd, w, dh=dh)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])  # the same bits
    only = tilec.ext.rms_norm_backward(dy, h, rstd, w, dh=dh, weight_grad=False)
    assert torch.equal(only[0], dx) and only[1] is None


def check_backward(dy, h, rstd, w, dh, dx, dw):
    R, D = h.shape
    dyd, r = dy.double(), rstd.double()[:, None]
    hhat = h.double() * r
    wdy = dyd if w is None else dyd * w.double()
    c = (wdy * hhat).mean(dim=1, keepdim=True)
    other = 0 if dh is None else dh.double()
    want = r * (wdy - hhat * c) + other
    # Every product and sum rounds once or twice; c carries its chain.
    tol = r * (wdy.abs() * 4 * E32 + hhat.abs() * (c.abs() * 6 * E32 + 90 * E32 * (wdy * hhat).abs().mean(dim=1, keepdim=True)))
    assert ((dx.double() - want).abs() <= tol + want.abs() * (half_ulp(dx.dtype) + 4 * E32) + 1e-37).all()
    wantw = (dyd * hhat).sum(dim=0)
    assert ((dw.double() - wantw).abs() <= (R + 64) * E32 * (dyd * hhat).abs().sum(dim=0) + 1e-37).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_views_and_missing_parameters(dt):
    # Rows of a wider matrix from an odd element on; parameters at odd elements.
    x, res, w = make(70, 333, dt, dt, dt)
    xv, rv, wv = x[:, 5:300], res[:, 3:298], w[1:296]
    for out in (None, torch.float8_e4m3fn):
        y, h, rstd = tilec.ext.rms_norm(xv, wv, rv, dtype=out)
        check_forward(xv, rv, wv, y, h, rstd)
    dy, dh = res[:, 7:302], x[:, 1:296]
    rstd = tilec.ext.rms_norm(xv)[2]
    check_backward(dy, xv, rstd, wv, dh, *tilec.ext.rms_norm_backward(dy, xv, rstd, wv, dh=dh))
    # Columns of a transposed matrix: copied.
    xt, rt = x.t()[:256], res.t()[:256]
    check_forward(xt, rt, None, *tilec.ext.rms_norm(xt, None, rt))
    # One row, one dimension; in 8 bits a row of its own.
    y, h, rstd = tilec.ext.rms_norm(x[4], w, res[4])
    assert y.shape == h.shape == (333,) and rstd.shape == (1,)
    check_forward(x[4:5], res[4:5], w, y[None], h[None], rstd)
    codes, scales = tilec.ext.rms_norm(x[4], w, res[4], dtype=torch.float8_e4m3fn)[0]
    assert codes.shape == (1, 333) and scales.shape == (1, 3)
    # A broadcast row: stride 0.
    xb = x[:1].expand(6, 333)
    check_forward(xb, None, w, *tilec.ext.rms_norm(xb, w))


@pytest.mark.gpu
def test_wide_row_stride():
    # Rows whose offsets pass 32 bits (in bytes).
    store = torch.empty((3, 1 << 29), dtype=torch.float32, device="cuda")
    x, res, w = make(3, 1000, "f32", "f32", "f32")
    v = store[:, :1000]
    v.copy_(x)
    y, h, rstd = tilec.ext.rms_norm(res, w, v)
    check_forward(res, v, w, y, h, rstd)
    check_backward(res, v, rstd, w, v, *tilec.ext.rms_norm_backward(res, v, rstd, w, dh=v))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # A matrix of more than 2^31 values, checked in its first and last rows.
    R, D = (1 << 19) + 3, 4096
    x = torch.empty((R, D), dtype=torch.bfloat16, device="cuda")
    x[:5], x[-5:] = make(5, D, "bf16")[0], make(5, D, "bf16", seed=1)[0]
    x[5:-5] = 1
    codes, scales = tilec.ext.rms_norm(x, dtype=torch.float8_e4m3fn)[0]
    y, _, rstd = tilec.ext.rms_norm(x)
    for rows in (slice(0, 5), slice(R - 5, R)):
        check_forward(x[rows], None, None, y[rows], x[rows], rstd[rows])
        check_forward(x[rows], None, None, (codes[rows], scales[rows]), x[rows], rstd[rows])
    dx, dw = tilec.ext.rms_norm_backward(y, x, rstd, dh=x)
    for rows in (slice(0, 5), slice(R - 5, R)):
        want = tilec.ext.rms_norm_backward(y[rows].clone(), x[rows].clone(), rstd[rows].clone(), dh=x[rows].clone())[0]
        assert torch.equal(dx[rows], want)


@pytest.mark.gpu
def test_special_values():
    # Rows of zeros: eps alone, codes of zero.
    z = torch.zeros((3, 200), device="cuda")
    y, h, rstd = tilec.ext.rms_norm(z, eps=1e-6)
    assert torch.equal(y, z) and torch.allclose(rstd, torch.full_like(rstd, 1e3))
    codes, scales = tilec.ext.rms_norm(z, eps=1e-6, dtype=torch.float8_e5m2)[0]
    assert torch.equal(codes.float(), z) and (scales == 2.0 ** -100 / 57344).all()
    # A row with an infinity or a NaN spoils that row and no other.
    x, _, w = make(9, 300, "f32")
    good = tilec.ext.rms_norm(x, w)[0]
    good8 = tilec.ext.dequantize_fp8(tilec.ext.rms_norm(x, w, dtype=torch.float8_e4m3fn)[0])
    x[3, 17], x[5, 299] = float("inf"), float("nan")
    y = tilec.ext.rms_norm(x, w)[0]
    y8 = tilec.ext.dequantize_fp8(tilec.ext.rms_norm(x, w, dtype=torch.float8_e4m3fn)[0])
    keep = [0, 1, 2, 4, 6, 7, 8]
    assert torch.equal(y[keep], good[keep]) and torch.equal(y8[keep], good8[keep])
    assert y[5].isnan().all() and y8[5].isnan().all() and y[3, 17].isnan() and y8[3, :128].isnan().all()


@pytest.mark.gpu
def test_no_rows():
    x = torch.empty((0, 40), device="cuda")
    y, h, rstd = tilec.ext.rms_norm(x, None, x)
    assert y.shape == h.shape == (0, 40) and rstd.shape == (0,)
    codes, scales = tilec.ext.rms_norm(x, dtype=torch.float8_e4m3fn)[0]
    assert codes.shape == (0, 40) and scales.shape == (0, 1)
    dx, dw = tilec.ext.rms_norm_backward(x, x, rstd, dh=x)
    assert dx.shape == (0, 40) and torch.equal(dw, torch.zeros(40, device="cuda"))


@pytest.mark.gpu
def test_gradients_against_differences():
    # Central differences of sum(dy * y) + sum(dh * h) in 64 bits; their own error is
    # step^2 times a third derivative, about 1e-8 here, and 2^-52 / step.
    x, dh, w = make(2, 13, "f32", "f32", seed=5)
    dy = torch.randn(2, 13, generator=torch.Generator().manual_seed(9)).cuda()
    _, h, rstd = tilec.ext.rms_norm(x, w)
    dx, dw = (t.cpu().double() for t in tilec.ext.rms_norm_backward(dy, h, rstd, w, dh=dh))
    x, dh, w, dy = (t.cpu().double() for t in (x, dh, w, dy))

    def f():
        return (dy * x * (x.square().mean(dim=1, keepdim=True) + 1e-5) ** -0.5 * w).sum() + (dh * x).sum()

    step = 1e-4
    for t, grad in ((x, dx), (w, dw)):
        flat, got = t.view(-1), grad.reshape(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + step
            up = f()
            flat[i] = keep - step
            down = f()
            flat[i] = keep
            assert abs((up - down) / (2 * step) - got[i]) <= 3e-6 * (1 + abs(got[i]))


@pytest.mark.gpu
def test_refusals():
    f, g = tilec.ext.rms_norm, tilec.ext.rms_norm_backward
    x, res, w = make(4, 8, "f32", "f32")
    stat = torch.zeros(4, device="cuda")
    for bad, error in (((x[None],), ValueError), ((x, w[:7]), ValueError), ((x, w, res[:3]), ValueError),
                       ((x, w, res.half()), TypeError), ((x.half(),), TypeError), ((x, w.half()), TypeError),
                       ((x, w, res.cpu()), TypeError), ((x, w.cpu()), TypeError), ((x, w, 3), TypeError),
                       ((torch.empty((3, 0), device="cuda"),), ValueError)):
        with pytest.raises(error):
            f(*bad)
    for dtype in (torch.float16, torch.int8, 8):
        with pytest.raises(TypeError):
            f(x, dtype=dtype)
    for bad, error in (((res[:3], x, stat), ValueError), ((res, x, stat[:3]), ValueError),
                       ((res, x, stat.double()), TypeError), ((res.double(), x, stat), TypeError),
                       ((res, x, stat, w[1:]), ValueError), ((res, x.cpu(), stat), TypeError),
                       ((res, x, stat, w, res[1:]), ValueError), ((res, x, stat, w, res.half()), TypeError)):
        with pytest.raises(error):
            g(*bad)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3)
    with pytest.raises(TypeError):
        tilec.ext.rms_norm(x)
    with pytest.raises(TypeError):
        tilec.ext.rms_norm_backward(x, x, torch.ones(2))


@pytest.mark.gpu
@pytest.mark.parametrize("ht,dt", [("f32", ""), ("f32", "f32"), ("bf16", ""), ("bf16", "bf16")])
@pytest.mark.parametrize("R,D", [(2, 4096), (130, 1600), (1023, 1009), (1024, 1009), (1025, 1009), (700, 2049), (1000, 40),
                                 (64, 16384), (257, 8200), (3, 15)])
def test_backward_of_few_rows(R, D, ht, dt):
    # Both gradients in one launch, several rows a workgroup, and just past that.
    h, dh, w = make(R, D, ht, dt, ht, seed=R * D)
    dy = torch.randn(R, D, generator=torch.Generator().manual_seed(R)).to(TYPES[ht]).cuda()
    rstd = tilec.ext.rms_norm(h, w)[2]
    dx, dw = tilec.ext.rms_norm_backward(dy, h, rstd, w, dh=dh)
    check_backward(dy, h, rstd, w, dh, dx, dw)
    again = tilec.ext.rms_norm_backward(dy, h, rstd, w, dh=dh)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@pytest.mark.gpu
def test_backward_of_few_rows_keeps_a_nan_to_its_row_and_column():
    h, _, w = make(300, 500, "f32", "", "f32", seed=8)
    dy = torch.randn(300, 500, generator=torch.Generator().manual_seed(9)).cuda()
    rstd = tilec.ext.rms_norm(h, w)[2]
    good = tilec.ext.rms_norm_backward(dy, h, rstd, w)
    dy[299, 499] = float("nan")
    dx, dw = tilec.ext.rms_norm_backward(dy, h, rstd, w)
    assert torch.equal(dx[:299], good[0][:299]) and dx[299].isnan().all()
    assert torch.equal(dw[:499], good[1][:499]) and dw[499].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,ht", [(1024, 4096, "f32"), (1024, 8192, "bf16"), (1000, 4001, "bf16"), (500, 512, "f32")])
def test_backward_of_the_largest_in_one_launch(R, D, ht):
    # Rows of whole lines, as a matrix of its own and as columns of a wider one.
    h, dh, w = make(R, D, ht, ht, ht, seed=R + D)
    dy = torch.randn(R, D, generator=torch.Generator().manual_seed(R)).to(TYPES[ht]).cuda()
    rstd = tilec.ext.rms_norm(h, w)[2]
    dx, dw = tilec.ext.rms_norm_backward(dy, h, rstd, w, dh=dh)
    check_backward(dy, h, rstd, w, dh, dx, dw)
    wide = torch.empty((R, D + 3), dtype=dy.dtype, device="cuda")
    wide[:, 2:D + 2] = dy
    again = tilec.ext.rms_norm_backward(wide[:, 2:D + 2], h, rstd, w, dh=dh)
    assert torch.equal(again[0], dx)
    check_backward(dy, h, rstd, w, dh, *again)
