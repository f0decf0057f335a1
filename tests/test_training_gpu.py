"""The training operators together: the example's training run, against the
same run in plain float32, and a step captured in a HIP graph."""

import math
import os
import sys

import pytest
import torch

import tilec

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import train_classifier as example  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_example_learns(bits):
    # Guessing costs log(1000); a tenth of the targets is noise, which costs at
    # least 0.1 log(1000) + H(0.1) = 1.02 per target to the best of models.
    losses, held_out = example.train(steps=80, tokens=2048, vocab=1000, width=64, hidden=128, bits=bits, log=None)
    assert abs(losses[0] - math.log(1000)) < 1.0
    assert held_out < 0.4 * math.log(1000) and losses[-1] < 0.4 * math.log(1000)


@pytest.mark.gpu
def test_one_step_against_plain_autograd():
    # One step of the example in torch's float32 autograd, on the same bf16
    # weights.  bf16 rounds the norm's output, dy, dh and the logits' gradient,
    # 2^-8 each at most, so the gradients agree to a few of those.
    follow = torch.randperm(500, generator=torch.Generator().manual_seed(1)).cuda()
    model = example.Model(500, 64, 96, 32)
    tokens, targets = example.batch(follow, 700, seed=3)
    w1, w, b, w2 = [c.float().requires_grad_() for c in model.copies]
    h = model.embedding[tokens].float() @ w1.t()
    y = torch.nn.functional.layer_norm(h, (96,), w, b)
    want = torch.nn.functional.cross_entropy(y @ w2.t(), targets, ignore_index=example.IGNORE)
    want.backward()
    x, hh, yy, mean, rstd = model.forward(tokens)
    loss, dy, dw2 = tilec.ext.linear_cross_entropy_grad(yy, model.copies[3], targets, ignore_index=example.IGNORE)
    dh, dw, db = tilec.ext.layer_norm_backward(dy, hh, mean, rstd, model.copies[1])
    dw1 = tilec.ext.matrix_mul(dh.t(), x)
    assert abs(loss.item() - want.item()) < 2e-3 * want.item()
    for got, grad in ((dw1, w1.grad), (dw, w.grad), (db, b.grad), (dw2, w2.grad)):
        assert (got.float() - grad).norm() <= 4 * 2.0 ** -8 * grad.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_graph_replays(dt):
    # Norm, loss with gradients, norm backward and optimizer in one graph,
    # replayed on new inputs with eager work in between; every replay against
    # the eager calls on the same inputs.
    g = torch.Generator(device="cuda").manual_seed(0)
    N, H, V = 300, 192, 1100
    x = torch.randn(N, H, generator=g, device="cuda").to(dt)
    w, b = torch.ones(H, device="cuda", dtype=dt), torch.zeros(H, device="cuda", dtype=dt)
    head = (torch.randn(V, H, generator=g, device="cuda") * 0.1).to(dt)
    t = torch.randint(V, (N,), generator=g, device="cuda")
    p = torch.randn(V, H, generator=g, device="cuda")

    def run(x, p, m, v):
        y, mean, rstd = tilec.ext.layer_norm(x, w, b)
        loss, dy, dhead = tilec.ext.linear_cross_entropy_grad(y, head, t)
        dx, dw, db = tilec.ext.layer_norm_backward(dy, x, mean, rstd, w)
        tilec.ext.adamw_step([p], [dhead], [m], [v], step=5)
        return loss, dx, dw, db

    m, v = tilec.ext.adamw_state(p, 8)
    start = [s.clone() for s in (p, *m, *v)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # scratch buffers stay in place from here on
        run(x, p, m, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run(x, p, m, v)
    for k in range(4):
        new = torch.randn(N, H, generator=g, device="cuda").to(dt)
        x.copy_(new)
        for s, value in zip((p, *m, *v), start):
            s.copy_(value)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in (*out, p, m[0], v[1])]
        q, m2, v2 = start[0].clone(), (start[1].clone(), start[2].clone()), (start[3].clone(), start[4].clone())
        want = (*run(new, q, m2, v2), q, m2[0], v2[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), k
