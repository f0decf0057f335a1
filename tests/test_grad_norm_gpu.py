"""The norm of a list of gradients and its clipping, against 64-bit sums.

The norm is a float64 sum rounded once, 2^-24 of itself (and the 64-bit oracle's
own additions, in another order, n 2^-53); the scale adds one rounding, a clipped
gradient the scale's and its own.
"""

import math

import pytest
import torch

import tilec

E32 = 2.0 ** -24
SIZES = [1, 3, 255, 4096, 4097, 0, 70001, 8, 131072, 5]


def grads(sizes, dtype, seed=0, std=1e-2, shift=0):
    """Gradients at any element alignment of one storage, nothing between them."""
    g = torch.Generator().manual_seed(seed)
    n = sum(sizes)
    flat = torch.randn(n + shift, generator=g).mul_(std).to(dtype).cuda()
    out, at = [], shift
    for k in sizes:
        out.append(flat[at:at + k])
        at += k
    return out


def norm64(gs):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in gs if g is not None))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_norm_and_scale(dtype, shift):
    gs = grads(SIZES, dtype, shift=shift)
    want = norm64(gs)
    for max_norm in (None, 0.5 * want, 2 * want, 0.0, math.inf):
        norm, scale = tilec.ext.grad_norm(gs, max_norm)
        assert norm.shape == scale.shape == () and norm.dtype == scale.dtype == torch.float32
        assert abs(norm.item() - want) <= 2 * E32 * want
        clip = 1.0 if max_norm is None else min(1.0, max_norm / (want + 1e-6))
        assert abs(scale.item() - clip) <= 2 * E32 * clip
        again = tilec.ext.grad_norm(gs, max_norm)
        assert torch.equal(norm, again[0]) and torch.equal(scale, again[1])  # the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("count,size", [(1, 1), (1, 3), (300, 100), (121, 5000), (240, 1), (3, 3000001)])
def test_many_tensors(count, size):
    a, b = grads([size] * count, torch.float32, seed=count), grads([size] * count, torch.bfloat16, seed=size)
    mixed = [x for pair in zip(a, b) for x in pair] + [None]
    want = norm64(mixed)
    norm, scale = tilec.ext.grad_norm(mixed, want / 3)
    assert abs(norm.item() - want) <= 2 * E32 * want
    before = [g.clone() for g in mixed[:-1]]
    assert torch.equal(tilec.ext.clip_grads(mixed, want / 3), norm)
    for g, old in zip(mixed, before):
        assert torch.equal(g, (old.float() * scale).to(g.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clip_in_place(dtype):
    store = torch.full((9000,), 7.0, dtype=dtype, device="cuda")
    gs = [store[1:4001], store[4005:4006], store[4100:8999]]
    for i, g in enumerate(grads([4000, 1, 4899], dtype, seed=2)):
        gs[i].copy_(g)
    before, want = store.clone(), norm64(gs)
    # Below the limit nothing is touched.
    norm = tilec.ext.clip_grads(gs, 1.5 * want)
    assert torch.equal(store, before) and abs(norm.item() - want) <= 2 * E32 * want
    scale = tilec.ext.grad_norm(gs, 0.25 * want)[1]
    tilec.ext.clip_grads(gs, 0.25 * want)
    expect = before.clone()
    for s in (slice(1, 4001), slice(4005, 4006), slice(4100, 8999)):
        expect[s] = (before[s].float() * scale).to(dtype)
    assert torch.equal(store, expect)  # and what lies between them stays
    # A factor of its own, above the limit and below it.
    factor = torch.tensor(0.125, device="cuda")
    norm, scale = tilec.ext.grad_norm(gs, 1e9, grad_scale=factor)
    assert scale.item() == 0.125 and abs(norm.item() - 0.125 * norm64(gs)) <= 4 * E32 * norm.item()
    expect = store.clone()
    tilec.ext.clip_grads(gs, 1e9, grad_scale=factor)
    assert torch.equal(gs[0], (expect[1:4001].float() * 0.125).to(dtype))
    norm, scale = tilec.ext.grad_norm(gs, 0.1 * norm64(gs), grad_scale=-torch.ones(1, device="cuda"))
    assert norm.item() > 0 and -0.11 < scale.item() < -0.09


@pytest.mark.gpu
def test_views():
    x = torch.randn(300, 200, device="cuda")
    want = norm64([x])
    for view in (x, x.t(), x.view(10, 30, 200).permute(2, 0, 1)):
        assert abs(tilec.ext.grad_norm([view])[0].item() - want) <= 2 * E32 * want
    half = x[:, ::2]  # read as a copy
    assert abs(tilec.ext.grad_norm([half])[0].item() - norm64([half])) <= 2 * E32 * want
    with pytest.raises(ValueError):
        tilec.ext.clip_grads([half], 1.0)
    old = x.clone()
    scale = tilec.ext.grad_norm([x.t()], 1.0)[1]
    tilec.ext.clip_grads([x.t()], 1.0)
    assert torch.equal(x, old * scale)
    # The same gradient twice counts twice, and is not multiplied twice.
    assert abs(tilec.ext.grad_norm([x, x])[0].item() - math.sqrt(2) * norm64([x])) <= 4 * E32
    for pair in ([x, x], [x[:10], x[9:20]], [x[0], x]):
        with pytest.raises(ValueError, match="share"):
            tilec.ext.clip_grads(pair, 1.0)
    tilec.ext.clip_grads([x[:10], x[10:]], 1.0)


@pytest.mark.gpu
def test_special_values():
    # Squares outside float32's range.
    for value in (1e30, 1e-30):
        x = torch.full((1000,), value, device="cuda")
        want = math.sqrt(1000) * x[0].item()
        norm, scale = tilec.ext.grad_norm([x], value)
        assert abs(norm.item() - want) <= 2 * E32 * want
        assert abs(scale.item() - min(1.0, value / (want + 1e-6))) <= 4 * E32
    x = torch.ones(1000, device="cuda")
    x[7] = float("inf")
    norm, scale = tilec.ext.grad_norm([x], 1.0)
    assert norm.item() == math.inf and scale.item() == 0
    x[8] = float("nan")
    norm, scale = tilec.ext.grad_norm([x], 1.0)
    assert math.isnan(norm.item()) and math.isnan(scale.item())
    zero = [torch.zeros(5, device="cuda"), torch.empty(0, device="cuda")]
    norm, scale = tilec.ext.grad_norm(zero, 1.0)
    assert norm.item() == 0 and scale.item() == 1
    norm, scale = tilec.ext.grad_norm(zero[1:], 1.0)
    assert norm.item() == 0 and scale.item() == 1
    assert tilec.ext.clip_grads(zero[1:], 1.0).item() == 0


@pytest.mark.gpu
def test_offsets_past_32_bits():
    n = (1 << 31) + 4099
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[:3], x[-5:] = 2, 3
    norm, scale = tilec.ext.grad_norm([x[1:]], 0.5)
    assert abs(norm.item() - math.sqrt(8 + 45)) <= 2 * E32 * 8
    tilec.ext.clip_grads([x[1:]], 0.5)
    want = (torch.tensor(3.0) * scale.cpu()).bfloat16()
    assert x[0].item() == 2 and (x[-5:].cpu() == want).all() and x[-6].item() == 0


@pytest.mark.gpu
def test_versions():
    # A backward pass that saved a gradient before it was clipped raises.
    w = torch.ones(4, device="cuda", requires_grad=True)
    g = torch.full((4,), 2.0, device="cuda")
    out = (w * g).sum()
    tilec.ext.grad_norm([g], 1.0)
    tilec.ext.clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="modified"):
        out.backward()


@pytest.mark.gpu
def test_with_adamw():
    # The scale as AdamW's factor steps as clipped gradients do, up to their rounding.
    gs = grads([5000, 33, 1], torch.float32, std=1.0)
    ps = [torch.randn(g.numel(), device="cuda") for g in gs]
    qs = [p.clone() for p in ps]

    def states():
        s = [tilec.ext.adamw_state(p) for p in ps]
        return [a for a, _ in s], [b for _, b in s]

    scale = tilec.ext.grad_norm(gs, 1.0)[1]
    tilec.ext.adamw_step(ps, gs, *states(), step=1, grad_scale=scale)
    tilec.ext.clip_grads(gs, 1.0)
    tilec.ext.adamw_step(qs, gs, *states(), step=1)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.gpu
def test_refusals():
    f, c = tilec.ext.grad_norm, tilec.ext.clip_grads
    x = torch.zeros(4, device="cuda")
    for bad, error in ((([],), ValueError), (([None],), ValueError), (([x.half()],), TypeError), (([x.cpu()],), TypeError),
                       (([x], -1.0), ValueError), (([x], math.nan), ValueError), (([x, 3],), TypeError), ((3,), TypeError),
                       (([x], 1.0, torch.ones(2, device="cuda")), ValueError), (([x], 1.0, torch.ones(1)), TypeError),
                       (([x], 1.0, torch.ones(1, device="cuda").double()), TypeError)):
        with pytest.raises(error):
            f(*bad)
        with pytest.raises(error):
            c(*(bad if len(bad) > 1 else (*bad, 1.0)))


def test_cpu_tensors_are_refused():
    x = torch.zeros(4)
    with pytest.raises(TypeError):
        tilec.ext.grad_norm([x])
    with pytest.raises(TypeError):
        tilec.ext.clip_grads([x], 1.0)


@pytest.mark.gpu
def test_an_infinite_limit_is_none():
    x = torch.ones(1000, device="cuda")
    x[7] = float("inf")
    norm, scale = tilec.ext.grad_norm([x], math.inf, grad_scale=torch.tensor(0.5, device="cuda"))
    assert norm.item() == math.inf and scale.item() == 0.5
    x[8] = float("nan")
    norm, scale = tilec.ext.grad_norm([x], math.inf)
    assert math.isnan(norm.item()) and scale.item() == 1
