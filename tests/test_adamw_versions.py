"""AdamW steps and autograd: what a step writes counts as modified in place."""

import pytest
import torch

import tilec


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_from_before_the_step_raises(bits):
    p = torch.randn(300, device="cuda", requires_grad=True)
    m, v = tilec.ext.adamw_state(p, bits)
    copy = p.detach().bfloat16().requires_grad_()
    g = torch.randn(300, device="cuda")
    losses = [p.square().sum(), copy.square().sum()]
    written = [p, copy, *((m, v) if bits == 32 else (*m, *v))]
    before, read = [t._version for t in written], g._version
    tilec.ext.adamw_step([p], [g], [m], [v], step=1, copies=[copy])
    assert all(t._version > b for t, b in zip(written, before)) and g._version == read
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # A graph from after it does not.
    p.square().sum().backward()
    assert torch.equal(p.grad, 2 * p.detach())


@pytest.mark.gpu
def test_refused_and_skipped_steps_leave_versions_alone():
    p, q = torch.randn(30, device="cuda"), torch.randn(30, device="cuda")
    g = torch.randn(30, device="cuda")
    s, t = tilec.ext.adamw_state(p), tilec.ext.adamw_state(q)
    before = [x._version for x in (p, *s, q, *t)]
    with pytest.raises(ValueError):
        tilec.ext.adamw_step([p], [g], [s[0]], [s[1]], step=1, lr=-1.0)
    with pytest.raises(ValueError):
        tilec.ext.adamw_step([p, q], [g, g[:3]], [s[0], t[0]], [s[1], t[1]], step=1)
    with pytest.raises(ValueError):
        tilec.ext.adamw_step([p], [g], [s[0]], [s[1]], step=1, grad_scale=torch.ones(2, device="cuda"))
    assert [x._version for x in (p, *s, q, *t)] == before
    tilec.ext.adamw_step([p, q], [g, None], [s[0], t[0]], [s[1], t[1]], step=1)
    assert [x._version for x in (q, *t)] == before[3:] and p._version > before[0]


@pytest.mark.gpu
def test_tensors_without_versions():
    with torch.inference_mode():
        p, g = torch.ones(10, device="cuda"), torch.ones(10, device="cuda")
        m, v = tilec.ext.adamw_state(p)
    tilec.ext.adamw_step([p], [g], [m], [v], step=1, lr=0.25, weight_decay=0.0)
    assert ((p - 0.75).abs() < 1e-6).all()


@pytest.mark.gpu
def test_lists_of_any_kind():
    p, g = torch.ones(10, device="cuda"), torch.ones(10, device="cuda")
    m, v = tilec.ext.adamw_state(p)
    tilec.ext.adamw_step(iter([p]), (g,), iter([m]), [v], step=1, lr=0.25, weight_decay=0.0)
    assert ((p - 0.75).abs() < 1e-6).all()
    with pytest.raises(TypeError):
        tilec.ext.adamw_step([p], [g], [m], [v], step=1.5)
    with pytest.raises(TypeError):
        tilec.ext.adamw_step([p], [g], [m], [v], step=1, grad_scale=0.5)
