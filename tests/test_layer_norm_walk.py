"""Layer norm where workgroups walk over rows: more rows than one step of the
grid takes, in every geometry (several rows side by side in a workgroup, one
row in a part of one, in a whole one, rows read more than once), with a last
step that is not full.  The plain 64-bit forms and the bounds are those of
test_layer_norm_gpu.

Rows of a step, at 256 CUs: 16 waves a CU forward, 8 (float32) or 12 (bfloat16)
backward; a row of D values has a power of two of threads up to a wave, whole
waves up to 1024 threads, with up to 16 values a thread (bfloat16 forward: 32).
The backward pass of rows over 16384 takes as many rows at a time as fill the
chip four times with 256-thread workgroups over the columns.
"""

import pytest
import torch

import tilec
from test_layer_norm_gpu import TYPES, check_backward, check_forward, make


@pytest.mark.gpu
@pytest.mark.parametrize("xt,yt,wt", [("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "bf16"),
                                      ("bf16", "f32", "f32")])
@pytest.mark.parametrize("R,D", [(4099, 3001), (140003, 64), (70001, 37), (9001, 700), (1300, 9216), (250, 20000)])
def test_rows_beyond_a_step_of_the_grid(R, D, xt, yt, wt):
    x, w, b, dy = make(R, D, xt, yt, wt, seed=R + D)
    x[-1] += 3.0  # the last row differs from the others
    y, mean, rstd = tilec.ext.layer_norm(x, w, b, dtype=TYPES[yt])
    check_forward(x, w, b, y, mean, rstd)
    dx, dw, db = tilec.ext.layer_norm_backward(dy, x, mean, rstd, w)
    check_backward(dy, x, mean, rstd, w, dx, dw, db)
    again = tilec.ext.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,D", [(4099, 3001), (140003, 64)])
def test_a_spoiled_row_stays_alone(R, D, dt):
    # What one step of a workgroup leaves behind must not reach its next rows.
    x, w, b, dy = make(R, D, dt, dt, dt, seed=3)
    want = tilec.ext.layer_norm(x, w, b)
    bad = x.clone()
    rows = [0, R // 2, R - 1]
    bad[rows[0], D - 1], bad[rows[1], 0], bad[rows[2], D // 2] = float("nan"), float("inf"), float("-inf")
    keep = torch.ones(R, dtype=torch.bool, device="cuda")
    keep[rows] = False
    got = tilec.ext.layer_norm(bad, w, b)
    assert all(torch.equal(p[keep], q[keep]) for p, q in zip(got, want)) and got[0][rows].isnan().all()
    dx = tilec.ext.layer_norm_backward(dy, x, want[1], want[2], w)[0]
    bad_dx = tilec.ext.layer_norm_backward(dy, bad, got[1], got[2], w)[0]
    assert torch.equal(dx[keep], bad_dx[keep]) and bad_dx[rows].isnan().all()
