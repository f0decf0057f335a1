"""Gradients of ignored rows are zeros whatever the gradient of the loss is: an
infinite one (an overflowed loss scale) or a NaN reaches the rows that count and
nothing else.
"""

import math

import pytest
import torch

import tilec


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,V,rows", [(20, 128, 1000, 0), (300, 136, 5003, 0), (300, 130, 1000, 100), (2304, 520, 16500, 0)])
def test_gradient_of_the_loss_that_is_not_finite(N, H, V, rows, dt, value):
    g = torch.Generator().manual_seed(N + V)
    x, w = torch.randn(N, H, generator=g).to(dt).cuda(), (torch.randn(V, H, generator=g) * 0.1).to(dt).cuda()
    t = torch.randint(V, (N,), generator=g).cuda()
    t[::3] = -100
    grad_loss = torch.tensor(value, device="cuda")
    for reduction in ("mean", "sum"):
        loss, dx, dw = tilec.ext.linear_cross_entropy_grad(x, w, t, reduction, grad_loss=grad_loss, chunk_rows=rows)
        assert loss.isfinite() and not dx[::3].any()
        assert not dx[1::3].isfinite().any() and not dw[t[t >= 0]].isfinite().any()
        none = torch.full_like(t, -100)
        loss, dx, dw = tilec.ext.linear_cross_entropy_grad(x, w, none, reduction, grad_loss=grad_loss, chunk_rows=rows)
        assert loss.item() == 0 and not dx.any() and not dw.any()
    each = torch.where(t == -100, value, 1.0)
    want = tilec.ext.linear_cross_entropy_grad(x, w, t, "none", chunk_rows=rows)
    got = tilec.ext.linear_cross_entropy_grad(x, w, t, "none", grad_loss=each, chunk_rows=rows)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and not got[1][::3].any()
