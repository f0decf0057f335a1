"""Every product of an 8-bit layer's step, as fp8.py's documentation writes the step
out, against the float64 product of the values that its operands' codes stand for; and
the step's gradients against float64 ones of the same layer.

Tolerances.  A product of operands given in 8 bits (S = sum |x| |w| of an output's
values): a float32 output adds 128 values a group, a group's sum to the other G, and up
to 64 splits' and waves' sums, each within 2^-24 of S.  A bfloat16 output's 8-bit
matrix instructions cut each product at 2^-13 of the power of two of the largest of
its eight: below 7 2^-13 of S in all, beside 2 2^-24 S for each of the 15 other eights
and the rounding of 2^-8 of the output.  Neither leaves room for a scale of another
block or a group of K that is missing: one of G groups is about 1 / G of S.

The whole step: a code is off by at most 2^-4 (e4m3) of its value.  Written as m 2^e
with 1 <= m < 2 it is off by d 2^e, d uniform in +-2^-4, so by 2^-4 / sqrt(3) of 2^e in
root mean square and less of the value: 0.58 of 2^-4 at most, for normal values.  Two operands
that are off independently join by squares.  n, rounded twice on its way into the
weight's gradient, adds its first rounding (and 2^-9 as a bfloat16) to both.  The
errors of K or R products have no common sign; 4 standard deviations of their sum
over an output of E values are 4 / sqrt(E) of it.
"""

import math

import pytest
import torch

import tilec

E32 = 2.0 ** -24
F8 = torch.float8_e4m3fn
RMS = 0.58 * 2.0 ** -4
SHAPES = [(9, 300, 130), (200, 384, 257), (700, 1024, 640), (300, 2048, 1030), (2100, 640, 2304)]


def make(R, D, H):
    g = torch.Generator(device="cuda").manual_seed(R)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    return {"x": normal(R, D).bfloat16(), "residual": normal(R, D, std=2.0).bfloat16(), "w": (1 + normal(D, std=0.1)).bfloat16(),
            "weight": normal(H, D, std=1 / math.sqrt(D)), "dy": normal(R, H).bfloat16(), "dh": normal(R, D).bfloat16()}


class Recorded:
    """tilec.ext, with every product's operands and result written down."""

    def __init__(self):
        self.products = []

    def __getattr__(self, name):
        return getattr(tilec.ext, name)

    def linear_fp8(self, x, weight, dtype=torch.float32):
        out = tilec.ext.linear_fp8(x, weight, dtype)
        self.products.append((x, weight, out))
        return out


def step(t):
    """The documented step."""
    doc = tilec.fp8.__doc__
    lines = doc[doc.index("A layer in 8 bits"):].splitlines()
    ext = Recorded()
    names = {"torch": torch, "tilec": type("tilec", (), {"ext": ext}), **t}
    exec("\n".join(line[4:] for line in lines if line.startswith("    ")), names)
    return names, ext.products


def values(q):
    codes, scales = q
    R, C = codes.shape
    block = 1 if scales.shape[0] == R else 128
    return codes.double() * scales.double().repeat_interleave(block, 0)[:R].repeat_interleave(128, 1)[:, :C]


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,H", SHAPES)
def test_every_product(R, D, H):
    _, products = step(make(R, D, H))
    assert [tuple(out.shape) for *_, out in products] == [(R, H), (R, D), (H, D)]
    for x, weight, out in products:
        xv, wv = values(x), values(weight).t().contiguous()
        want, S = torch.mm(xv, wv), torch.mm(xv.abs(), wv.abs())
        G = -(-xv.shape[1] // 128)
        tol = (128 + G + 64) * E32 * S + 2 * E32 * want.abs()
        if out.dtype == torch.bfloat16:
            tol += 7 * 2.0 ** -13 * S + 2.0 ** -8 * want.abs()
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,H", SHAPES)
def test_gradients_of_the_layer(R, D, H):
    t = make(R, D, H)
    got, _ = step(t)
    h = (t["x"].float() + t["residual"].float()).bfloat16().double().requires_grad_()
    w, W = t["w"].double().requires_grad_(), t["weight"].double().requires_grad_()
    n = h * (h.square().mean(dim=1, keepdim=True) + 1e-5) ** -0.5 * w
    y = n @ W.t()
    (y * t["dy"].double()).sum().backward()

    def off(a, b):
        return ((a.double() - b).norm() / b.norm()).item()

    def most(*parts, of):
        return math.hypot(*parts) * (1 + 4 / math.sqrt(of))

    half = 2.0 ** -8  # bfloat16, at most
    assert off(got["y"], y) <= most(RMS, RMS, half, of=R * H)
    assert off(got["dn"], t["dy"].double() @ W.detach()) <= most(RMS, RMS, half, of=R * D)
    assert off(got["dweight"], W.grad) <= most(RMS, RMS, RMS, half, of=H * D)
    # dx - dh: dn's error, which the norm's gradient weighs as it weighs dn, and the
    # rounding of dx, which has dh in it.
    rest = got["dx"].double() - t["dh"].double()
    rounding = half * (got["dx"].double().norm() / h.grad.norm()).item()
    assert off(rest, h.grad) <= most(RMS, RMS, half, of=R * D) + rounding
    assert off(got["dw"], w.grad) <= most(RMS, RMS, half, of=D)

