"""Where the C entry points of the RMS norm allow an output in an input's place, the
results are those of separate outputs, bit for bit: dx in dh's place, h in the
residual's.  (tilec.ext allocates every output, so nothing there gets here.)"""

import pytest
import torch

import tilec
from tilec import _lib

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODE = {"f32": _lib.F32, "bf16": _lib.BF16}
E4 = torch.float8_e4m3fn


def normal(R, D, dtype, seed, wide=0):
    """[R, D], rows `wide` more values apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(R, D + wide, generator=g, device="cuda").to(TYPES[dtype])[:, :D]


def backward(dy, h, rstd, w, dh, dx, dw, names):
    R, D = h.shape
    L = _lib.lib()
    need = L.tilec_rms_norm_backward_workspace_bytes(R, D, CODE[names[1]])
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    _lib.check(L.tilec_rms_norm_backward(
        dy.data_ptr(), h.data_ptr(), rstd.data_ptr(), w.data_ptr(), dh.data_ptr(), dx.data_ptr(),
        None if dw is None else dw.data_ptr(), R, D, dy.stride(0), h.stride(0), dh.stride(0), dx.stride(0), CODE[names[0]],
        CODE[names[1]], CODE[names[2]], _lib.F32, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()


# One launch for both gradients, two, and rows that no workgroup holds.
@pytest.mark.gpu
@pytest.mark.parametrize("dyt,ht,dht", [("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "bf16"),
                                        ("bf16", "f32", "f32"), ("bf16", "bf16", "f32")])
@pytest.mark.parametrize("R,D", [(64, 4096), (1000, 1009), (2, 64), (3000, 512), (1, 300), (5, 20000), (40, 33333)])
def test_dx_in_the_place_of_dh(R, D, dyt, ht, dht):
    dy, h, dh = normal(R, D, dyt, 1), normal(R, D, ht, 2, 3), normal(R, D, dht, 3, 5)
    w = normal(1, D, "f32", 4)[0].contiguous()
    rstd = torch.rand(R, device="cuda") + 0.5
    for sums in (True, False):
        apart, dw = torch.empty(R, D, dtype=dh.dtype, device="cuda"), torch.empty(D, device="cuda") if sums else None
        backward(dy, h, rstd, w, dh, apart, dw, (dyt, ht, dht))
        place = torch.empty_strided(dh.shape, dh.stride(), dtype=dh.dtype, device="cuda").copy_(dh)
        dw2 = torch.empty(D, device="cuda") if sums else None
        backward(dy, h, rstd, w, place, place, dw2, (dyt, ht, dht))
        assert torch.equal(place, apart)
        assert not sums or torch.equal(dw, dw2)


def forward(x, res, w, y, ys, h, rstd, xt, rt):
    R, D = x.shape
    yt = _lib.F8E4M3 if ys is not None else CODE[xt]
    _lib.check(_lib.lib().tilec_rms_norm(
        x.data_ptr(), res.data_ptr(), w.data_ptr(), y.data_ptr(), None if ys is None else ys.data_ptr(), h.data_ptr(),
        rstd.data_ptr(), R, D, x.stride(0), res.stride(0), y.stride(0), h.stride(0), 0 if ys is None else ys.stride(0),
        0 if ys is None else ys.stride(1), CODE[xt], CODE[rt], yt, _lib.F32, 1e-5, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("xt,rt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("R,D", [(1, 4096), (7, 300), (2500, 129), (33, 16384), (3, 20000), (5, 40001)])
@pytest.mark.parametrize("bits8", [False, True])
def test_h_in_the_place_of_the_residual(R, D, xt, rt, bits8):
    x, res = normal(R, D, xt, 1, 3), normal(R, D, rt, 2, 5)
    w = normal(1, D, "f32", 4)[0].contiguous()

    def run(res, h):
        room = -(-D // 16) * 16
        y = torch.zeros(R, room if bits8 else D, dtype=torch.uint8 if bits8 else TYPES[xt], device="cuda")
        ys = torch.zeros(R, -(-D // 128), device="cuda") if bits8 else None
        rstd = torch.zeros(R, device="cuda")
        forward(x, res, w, y, ys, h, rstd, xt, rt)
        return [t for t in (y, ys, rstd) if t is not None]

    apart = torch.empty(R, D, dtype=res.dtype, device="cuda")
    want = run(res, apart)
    place = torch.empty_strided(res.shape, res.stride(), dtype=res.dtype, device="cuda").copy_(res)
    got = run(place, place)
    assert torch.equal(place, apart) and all(torch.equal(a, b) for a, b in zip(got, want))
