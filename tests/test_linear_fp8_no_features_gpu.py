"""Products of no features are zeros, also where there are more outputs than one grid of
tiles holds, and nothing but the outputs is written."""

import pytest
import torch

import tilec
from tilec import _lib

CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,ldo", [(1, 1, 1), (1, 300, 300), (300, 1, 1), (129, 257, 257), (129, 257, 300), (5000, 3, 5),
                                     (3, 70001, 70002)])
def test_rows_of_zeros(M, N, ldo, dtype):
    out = torch.ones(M, ldo, dtype=dtype, device="cuda")
    _lib.check(_lib.lib().tilec_linear_fp8(None, None, None, None, out.data_ptr(), M, N, 0, 0, 0, ldo, 0, 0, 0, 0, _lib.F8E4M3,
                                           _lib.F8E5M2, CODE[dtype], 1, 128, None, 0, None, 0,
                                           torch.cuda.current_stream().cuda_stream))
    assert (out[:, :N] == 0).all() and (out[:, N:] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1 << 30, 1), (1, (1 << 31) - 1024)])
def test_more_outputs_than_tiles(M, N):
    # (Whatever the allocator hands out was written before: not zeros by chance.)
    torch.full((M * N,), 1.0, dtype=torch.bfloat16, device="cuda")
    x, w = (torch.empty((R, 0), dtype=torch.float8_e4m3fn, device="cuda") for R in (M, N))
    sx, sw = (torch.empty((R, 0), device="cuda") for R in (M, N))
    out = tilec.ext.linear_fp8((x, sx), (w, sw), dtype=torch.bfloat16)
    assert out.shape == (M, N) and not out.any()


@pytest.mark.gpu
def test_in_a_graph():
    x, w = (torch.empty((R, 0), dtype=torch.float8_e4m3fn, device="cuda") for R in (70, 90))
    sx, sw = (torch.empty((R, 0), device="cuda") for R in (70, 90))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tilec.ext.linear_fp8((x, sx), (w, sw))
    for _ in range(4):
        out.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert not out.any() and not tilec.ext.linear_fp8((x, sx), (w, sw)).any()
