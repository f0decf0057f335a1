"""Outputs of the RMS norm's C entry points in the place of an input that is read after
they are written: refused before anything is enqueued (no GPU is needed).  Where an
output may be in an input's place, with the rows of both where they are, is in
test_rms_norm_in_place_gpu.py."""

import pytest

from tilec import _lib

F32, BF16 = _lib.F32, _lib.BF16


def backward(dy=1 << 20, h=2 << 20, dh=None, dx=3 << 20, R=4, D=64, lddy=64, ldh=64, lddh=64, lddx=64, t=F32, dw=4 << 20):
    return _lib.lib().tilec_rms_norm_backward(dy, h, 5 << 20, None, dh, dx, dw, R, D, lddy, ldh, lddh, lddx, t, t, t, F32, None,
                                              0, None)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("R,D", [(1, 64), (64, 4096), (1000, 1009), (3000, 512), (5, 20000)])
@pytest.mark.parametrize("dw", [None, 4 << 20])
def test_dx_in_the_place_of_dy_or_h(R, D, t, dw):
    ld = dict(R=R, D=D, lddy=D, ldh=D, lddh=D, lddx=D, t=t, dw=dw)
    assert backward(dx=1 << 20, **ld) == _lib.ERR_VALUE and "dx is dy" in _lib.last_error()
    assert backward(dx=2 << 20, **ld) == _lib.ERR_VALUE and "dx is h" in _lib.last_error()
    assert backward(dx=2 << 20, dh=6 << 20, **ld) == _lib.ERR_VALUE and "dx is h" in _lib.last_error()
    assert dw is not None or backward(dx=2 << 20, R=0, dw=None) == _lib.OK  # no rows: nothing is written


def test_in_the_place_of_an_input_but_with_other_rows():
    both = dict(dx=6 << 20, dh=6 << 20)
    assert backward(lddx=64, lddh=65, **both) == _lib.ERR_VALUE and "dx is dh" in _lib.last_error()
    assert backward(lddx=80, lddh=64, **both) == _lib.ERR_VALUE and "dx is dh" in _lib.last_error()

    def forward(ldr, ldh):
        return _lib.lib().tilec_rms_norm(1 << 20, 2 << 20, None, 3 << 20, None, 2 << 20, None, 4, 64, 64, ldr, 64, ldh, 0, 0, F32,
                                         F32, F32, F32, 1e-5, None)

    for ldr, ldh in ((64, 65), (80, 64)):
        assert forward(ldr, ldh) == _lib.ERR_VALUE and "h is the residual" in _lib.last_error()
