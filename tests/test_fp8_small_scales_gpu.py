"""Products of operands whose scales are small, large, or both: the product of two
scales is one float32, so it is off by 2^-24 of itself, and by 2^-150 where it is below
2^-126.  P, a group's sum of products of codes, is multiplied by it: beside a
product's other roundings (test_fp8_gpu.py) an output is off by 2^-150 of the sum of
its groups' |P|, and its own sums and rounding have steps of 2^-149 (bfloat16 2^-133)
below the normal range."""

import pytest
import torch

import tilec

E32 = 2.0 ** -24
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
WIDE = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = [(1, 100, 300), (12, 130, 513), (40, 300, 2100), (300, 200, 256), (700, 600, 384), (2100, 2300, 130)]


def operand(R, C, to, block, at, seed):
    """Codes over the range, scales of 2^at to 2^(at + 1)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    top = torch.finfo(F8[to]).max
    room = -(-C // 16) * 16
    codes = (torch.randn(R, room, generator=g, device="cuda") * top / 4).clamp(-top, top).to(F8[to])[:, :C]
    scales = torch.rand(-(-R // block), -(-C // 128), generator=g, device="cuda") + 1
    return codes, scales * 2.0 ** at


def expand(scales, block, R, C):
    return scales.double().repeat_interleave(block, 0)[:R].repeat_interleave(128, 1)[:, :C]


@pytest.mark.gpu
@pytest.mark.parametrize("xt,wt", [("e4m3", "e4m3"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("xat,wat", [(-75, -75), (-63, -63), (-70, -80), (-63, -85), (100, -100), (-110, 110), (-90, -50)])
@pytest.mark.parametrize("wb", [1, 128])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_scales(xt, wt, xat, wat, wb, out):
    for M, N, K in SIZES:
        x, w = operand(M, K, xt, 1, xat, M), operand(N, K, wt, wb, wat, N)
        got = tilec.ext.linear_fp8(x, w, dtype=WIDE[out]).double()
        xc, wc = x[0].double(), w[0].double().t().contiguous()
        xv, wv = xc * expand(x[1], 1, M, K), wc * expand(w[1], wb, N, K).t()
        want, S, P = torch.mm(xv, wv), torch.mm(xv.abs(), wv.abs()), torch.mm(xc.abs(), wc.abs())
        G = -(-K // 128)
        tol = (128 + G + 16) * E32 * S + 2 * E32 * want.abs() + 2.0 ** -150 * P + (G + 16) * 2.0 ** -149
        if out == "bf16":
            tol += 7 * 2.0 ** -13 * S + 2.0 ** -8 * want.abs() + 2.0 ** -134
        assert torch.isfinite(got).all() and ((got - want).abs() <= tol).all(), (M, N, K)
