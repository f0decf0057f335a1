"""AdamW's lists and the memory behind them: what would be written twice in one
step is refused, whatever offsets it starts at.
"""

import pytest
import torch

import tilec


def lists(sizes, bits=32, dtype=torch.float32):
    P = [torch.randn(n, device="cuda").to(dtype) for n in sizes]
    G = [torch.randn(n, device="cuda") for n in sizes]
    states = [tilec.ext.adamw_state(p, bits) for p in P]
    return P, G, [s[0] for s in states], [s[1] for s in states]


@pytest.mark.gpu
def test_overlapping_memory_is_refused():
    step = tilec.ext.adamw_step
    flat = torch.zeros(4096, device="cuda")
    half = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    P, G, M, V = lists([1000, 1000, 300])
    for at in range(4):  # params, grads, exp_avg, exp_avg_sq
        args = [list(a) for a in (P, G, M, V)]
        args[at][0], args[at][1] = flat[:1000], flat[999:1999]
        if at == 1:  # two gradients may be one memory, or overlap: they are read only
            step(*args, step=1)
            args[1][1] = args[1][0]
            step(*args, step=2)
            continue
        with pytest.raises(ValueError, match="share"):
            step(*args, step=1)
        args[at][1] = flat[1000:2000]  # next to each other
        step(*args, step=1)
        args[at][1] = args[at][0]
        with pytest.raises(ValueError, match="share"):
            step(*args, step=1)
    # Among kinds: a state in another parameter's memory, a gradient in a state's.
    with pytest.raises(ValueError, match="share"):
        step([flat[:1000], P[1]], G[:2], M[:2], [V[0], flat[900:1900]], step=1)
    with pytest.raises(ValueError, match="share"):
        step(P[:2], [flat[:1000], G[1]], M[:2], [V[0], flat[10:1010]], step=1)
    with pytest.raises(ValueError, match="share"):  # its own, but not value by value
        step([flat[:1000]], [flat[1:1001]], M[:1], V[:1], step=1)
    # Copies.
    with pytest.raises(ValueError, match="share"):
        step(P, G, M, V, step=1, copies=[half[:1000], half[500:1500], None])
    with pytest.raises(ValueError, match="share"):
        step(P, G, M, V, step=1, copies=[half[:1000], None, half[:300]])
    step(P, G, M, V, step=1, copies=[half[:1000], half[1000:2000], half[2000:2300]])


@pytest.mark.gpu
def test_overlapping_states_of_8_bits_are_refused():
    step = tilec.ext.adamw_step
    P, G, M, V = lists([1000, 1000], 8)
    for at, k in ((2, 0), (2, 1), (3, 0), (3, 1)):  # codes and scales of each state
        args = [P, G, list(M), list(V)]
        pair = list(args[at][1])
        pair[k] = args[at][0][k]
        args[at][1] = tuple(pair)
        with pytest.raises(ValueError, match="share"):
            step(*args, step=1)
    step(P, G, M, V, step=1)


@pytest.mark.gpu
def test_results_in_the_place_of_what_they_come_from():
    # Every value is read by the thread that writes it, so these are sound.
    P, G, M, V = lists([1000, 300], dtype=torch.bfloat16)
    G = [g.bfloat16() for g in G]
    want = [[t.clone() for t in a] for a in (P, G, M, V)]
    tilec.ext.adamw_step(*want, step=1)
    copies = [P[0], G[1]]
    tilec.ext.adamw_step(P, G, M, V, step=1, copies=copies)
    assert all(torch.equal(a, b) for a, b in zip(P, want[0]))
    assert all(torch.equal(a, b) for a, b in zip(copies, want[0]))
    assert all(torch.equal(a, b) for a, b in zip(M + V, want[2] + want[3]))


@pytest.mark.gpu
def test_empty_tensors_share_nothing():
    P, G, M, V = lists([0, 0, 5])
    tilec.ext.adamw_step([P[0], P[0], P[2]], [G[0], G[0], G[2]], [M[0], M[0], M[2]], [V[0], V[0], V[2]], step=1)
