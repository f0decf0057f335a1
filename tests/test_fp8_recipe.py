"""The 8-bit layer that fp8.py's documentation writes out, run as it stands there with
plain float64 operators in the place of the package's, against autograd."""

import types

import torch

import tilec

EPS = 1e-5


def recipe():
    """The documentation's lines of code, from where the layer begins."""
    doc = tilec.fp8.__doc__
    lines = doc[doc.index("A layer in 8 bits"):].splitlines()
    return "\n".join(line[4:] for line in lines if line.startswith("    "))


def rms_norm(x, weight=None, residual=None, eps=EPS, dtype=None):
    h = x + residual
    rstd = (h.square().mean(dim=1) + eps) ** -0.5
    return (h * rstd[:, None] * weight,), h, rstd  # a tuple: 8 bits are no matrix


def rms_norm_backward(dy, h, rstd, weight=None, dh=None):
    hhat = h * rstd[:, None]
    wdy = dy * weight
    dx = rstd[:, None] * (wdy - hhat * (wdy * hhat).mean(dim=1, keepdim=True))
    return dx + (0 if dh is None else dh), (dy * hhat).sum(dim=0)


def plain():
    return types.SimpleNamespace(
        rms_norm=rms_norm, rms_norm_backward=rms_norm_backward, quantize_fp8=lambda x, block=None, dtype=None: (x,),
        dequantize_fp8=lambda q, dtype=None: q[0], linear_fp8=lambda x, w, dtype=None: x[0] @ w[0].t())


def test_gradients_of_the_documented_layer():
    g = torch.Generator().manual_seed(0)
    x, residual, dh = (torch.randn(9, 20, generator=g, dtype=torch.float64) for _ in range(3))
    w, weight = 1 + 0.1 * torch.randn(20, generator=g, dtype=torch.float64), torch.randn(7, 20, generator=g, dtype=torch.float64)
    dy = torch.randn(9, 7, generator=g, dtype=torch.float64)
    names = {"torch": torch, "tilec": types.SimpleNamespace(ext=plain()), **vars(plain()), "x": x, "residual": residual, "w": w,
             "weight": weight, "dy": dy, "dh": dh}
    exec(recipe(), names)
    xa, ra, wa, Wa = (t.clone().requires_grad_() for t in (x, residual, w, weight))
    h = xa + ra
    y = h * (h.square().mean(dim=1, keepdim=True) + EPS) ** -0.5 * wa @ Wa.t()
    ((y * dy).sum() + (h * dh).sum()).backward()
    for name, want in (("y", y), ("dx", xa.grad), ("dx", ra.grad), ("dw", wa.grad), ("dweight", Wa.grad)):
        assert name in names, f"no {name}"
        assert torch.allclose(names[name], want.detach(), rtol=1e-10, atol=1e-12), name
