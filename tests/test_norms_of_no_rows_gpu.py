"""Gradients of parameters over no rows: zeros, however many columns there are."""

import pytest
import torch

import tilec


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 300, 20000, 1 << 26, (1 << 26) + 7])
def test_rms_norm(D, dtype):
    none = torch.empty((0, D), dtype=dtype, device="cuda")
    rstd = torch.empty(0, device="cuda")
    torch.full((D,), 1.0, device="cuda")  # (what the allocator hands out next: not zeros by chance)
    dx, dw = tilec.ext.rms_norm_backward(none, none, rstd)
    assert dx.shape == (0, D) and dw.shape == (D,) and dw.dtype == torch.float32 and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 300, 20000, 1 << 25, (1 << 26) + 7])
def test_layer_norm(D, dtype):
    none = torch.empty((0, D), dtype=dtype, device="cuda")
    stats = torch.empty(0, device="cuda")
    torch.full((2 * D,), 1.0, device="cuda")
    dx, dw, db = tilec.ext.layer_norm_backward(none, none, stats, stats)
    assert dx.shape == (0, D)
    for sums in (dw, db):
        assert sums.shape == (D,) and sums.dtype == torch.float32 and not sums.any()
