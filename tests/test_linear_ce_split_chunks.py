"""Linear cross entropy in chunks of rows whose weight gradient also splits the
rows of a chunk: the splits are joined onto what earlier chunks left, and a last
chunk that is too short to be split adds its own.  Plain forms and bounds are
those of test_linear_ce_gpu.
"""

import ctypes

import pytest
import torch

import tilec
from test_linear_ce_gpu import check, make
from tilec import _lib


def cdiv(a, b):
    return -(-a // b)


def split_bytes(x, w, rows):
    """Bytes of the workspace that hold the sums of K splits: what is left of it
    beside everything else (mean, gradients, bfloat16, operands read in place)."""
    (N, H), V = x.shape, w.shape[0]
    ws, cnt, got = ctypes.c_size_t(0), ctypes.c_size_t(0), ctypes.c_int64(0)
    _lib.check(_lib.lib().tilec_linear_ce_scratch_bytes(x.data_ptr(), w.data_ptr(), N, H, V, H, H, _lib.BF16, 2, 1, rows,
                                                        None, ctypes.byref(ws), ctypes.byref(cnt), ctypes.byref(got)))
    assert got.value == rows
    parts = [rows * cdiv(V, 256) * 4 * 8, rows * 4, N * 4, 4, rows * cdiv(H, 64) * 64 * 2, rows * cdiv(V, 64) * 64 * 2,
             V * cdiv(H, 16) * 16 * 4]
    return ws.value - sum(cdiv(p, 256) * 256 for p in parts)


@pytest.mark.gpu
@pytest.mark.parametrize("N,H,V,rows", [(9000, 72, 1001, 4099),  # 13 splits each, the last chunk shorter
                                        (8238, 72, 1001, 4099),  # a last chunk of 40 rows: one K step, no split
                                        (9000, 200, 500, 3000), (9000, 520, 3000, 4099)])
def test_split_weight_gradients_over_chunks(N, H, V, rows):
    x, w, t = make(N, H, V, "bf16", seed=N + V, ignored=0.2)
    assert split_bytes(x, w, rows) >= 2 * V * cdiv(H, 16) * 16 * 4  # dW splits K
    got = check(x, w, t, chunk_rows=rows)
    assert all(torch.equal(a, b) for a, b in zip(got, tilec.ext.linear_cross_entropy_grad(x, w, t, chunk_rows=rows)))
    g = torch.Generator().manual_seed(4)
    check(x, w, t, "none", torch.randn(N, generator=g).cuda(), chunk_rows=rows)
