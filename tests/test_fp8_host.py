"""What the entry points of the 8-bit operators, the RMS norm and the gradient norm
refuse before anything reaches a GPU (none is needed here), and the workspace that
they ask for."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch

import tilec
from tilec import _lib

F32, BF16, E4, E5 = _lib.F32, _lib.BF16, _lib.F8E4M3, _lib.F8E5M2
OK, VALUE, TYPE, WORKSPACE = _lib.OK, _lib.ERR_VALUE, _lib.ERR_TYPE, _lib.ERR_WORKSPACE


def linear(M=4, N=8, K=256, x=16, sx=16, w=16, sw=16, out=16, ldx=None, ldw=None, ldo=None, srow=2, sgroup=1, xd=E4, wd=E5,
           od=F32, xb=1, wb=128, ws=None, ws_bytes=0, cnt=None, cnt_bytes=0):
    # Non-null dummy pointers: every case must fail (or finish) before launch.
    return _lib.lib().tilec_linear_fp8(x, sx, w, sw, out, M, N, K, K if ldx is None else ldx, K if ldw is None else ldw,
                                       N if ldo is None else ldo, srow, sgroup, 2, 1, xd, wd, od, xb, wb, ws, ws_bytes, cnt,
                                       cnt_bytes, None)


def linear_bytes(M, N, K, x=16, w=16, ldx=None, ldw=None, od=F32):
    ws, cnt = ctypes.c_size_t(), ctypes.c_size_t()
    rc = _lib.lib().tilec_linear_fp8_scratch_bytes(x, w, M, N, K, K if ldx is None else ldx, K if ldw is None else ldw, E4, E4,
                                                   od, ctypes.byref(ws), ctypes.byref(cnt))
    assert rc == OK and cnt.value % 256 == 0 and (cnt.value == 0 or ws.value > 0)
    return ws.value


def test_linear_refusals():
    for kw in ({"xd": F32}, {"wd": BF16}, {"od": E4}, {"od": 7}, {"xd": -1}):
        assert linear(**kw) == TYPE, kw
    for kw in ({"M": -1}, {"K": -1}, {"N": 1 << 31}, {"K": (1 << 22) + 1}, {"ldx": 255}, {"ldw": 255}, {"ldo": 7},
               {"ldx": 1 << 41}, {"xb": 2}, {"wb": 0}, {"x": None}, {"sx": None}, {"w": None}, {"sw": None}, {"out": None},
               {"srow": -1}, {"srow": (1 << 21) + 1}, {"sgroup": -1}):
        assert linear(**kw) == VALUE, kw
        assert "linear_fp8" in _lib.last_error()
    assert linear(M=0, x=None, out=None) == OK and linear(N=0, w=None, out=None) == OK
    # An unaligned operand is copied, split sums are kept.
    assert linear(x=17) == WORKSPACE and linear(ldw=257) == WORKSPACE
    assert linear(M=100, N=100, K=8192) == WORKSPACE and linear(M=100, N=100, K=8192, ws=16, ws_bytes=1000) == WORKSPACE
    need = linear_bytes(100, 100, 8192)
    assert linear(M=100, N=100, K=8192, ws=16, ws_bytes=need) == WORKSPACE and "counter" in _lib.last_error()
    assert linear(M=100, N=100, K=8192, ws=16, ws_bytes=need, cnt=16, cnt_bytes=255) == WORKSPACE


def test_linear_workspace():
    assert linear_bytes(1, 4096, 4096) == 0 and linear_bytes(8192, 8192, 8192, od=BF16) == 0
    # 130 is no multiple of 16: both operands are copied, whatever x's address.
    assert linear_bytes(5, 7, 130, x=17) == linear_bytes(5, 7, 130, ldx=130) == 5 * 144 + 7 * 144
    assert linear_bytes(5, 7, 130, x=17, ldw=144) == 5 * 144
    assert linear_bytes(1, 7, 128, ldx=3) == 0  # one row has no stride
    assert linear_bytes(5, 7, 128, w=24) == 7 * 128
    assert linear_bytes(100, 100, 8192) % (128 * 128 * 4) == 0 and linear_bytes(100, 100, 8192) >= 2 * 100 * 100 * 4
    assert linear_bytes(0, 7, 130, x=17) == linear_bytes(5, 7, 0) == 0
    assert _lib.lib().tilec_linear_fp8_scratch_bytes(16, 16, -1, 7, 130, 130, 130, E4, E4, F32, None, None) == VALUE


def test_quantize_refusals():
    def q(R=4, C=256, x=16, codes=16, scales=16, ldx=None, ldq=256, srow=2, sgroup=1, layout=0, xd=F32, qd=E4, block=1):
        return _lib.lib().tilec_quantize_fp8(x, codes, scales, R, C, (R if layout else C) if ldx is None else ldx, ldq, srow,
                                             sgroup, layout, xd, qd, block, None)

    for kw in ({"xd": E4}, {"qd": F32}):
        assert q(**kw) == TYPE, kw
    for kw in ({"R": -1}, {"C": 1 << 31}, {"block": 64}, {"layout": 2}, {"ldx": 255}, {"ldx": 3, "layout": 1}, {"ldq": 264},
               {"ldq": 240}, {"codes": 24}, {"x": None}, {"codes": None}, {"scales": None}, {"srow": -1}):
        assert q(**kw) == VALUE, kw
    assert q(R=0, x=None) == OK and q(C=0, x=None, ldq=0) == OK

    def d(R=4, C=256, codes=16, scales=16, out=16, ldq=256, ldo=256, qd=E4, od=F32, block=1):
        return _lib.lib().tilec_dequantize_fp8(codes, scales, out, R, C, ldq, ldo, 2, 1, qd, od, block, None)

    assert d(qd=F32) == TYPE and d(od=E5) == TYPE
    for kw in ({"R": -1}, {"ldq": 255}, {"ldo": 255}, {"block": 3}, {"codes": None}, {"scales": None}, {"out": None}):
        assert d(**kw) == VALUE, kw
    assert d(R=0, codes=None) == OK


def test_rms_refusals():
    def f(R=4, D=64, x=16, res=None, w=None, y=16, ys=None, h=None, ldx=64, ldr=64, ldy=64, ldh=64, xd=F32, rd=F32, yd=F32, wd=F32):
        return _lib.lib().tilec_rms_norm(x, res, w, y, ys, h, None, R, D, ldx, ldr, ldy, ldh, 1, 1, xd, rd, yd, wd, 1e-5, None)

    for kw in ({"xd": E4}, {"yd": 9}, {"wd": E5}, {"rd": E4, "res": 16, "h": 16}):
        assert f(**kw) == TYPE, kw
    for kw in ({"R": -1}, {"D": 0}, {"x": None}, {"y": None}, {"ldx": 63}, {"ldy": 63}, {"res": 16}, {"res": 16, "h": 16, "ldr": 3},
               {"res": 16, "h": 16, "ldh": 3}, {"yd": E4}, {"yd": E4, "ys": 16, "y": 24}, {"yd": E4, "ys": 16, "ldy": 72}):
        assert f(**kw) == VALUE, kw
    assert f(R=0, x=None, y=None) == OK
    L = _lib.lib()

    def b(R=4, D=64, dy=16, h=16, rstd=16, dh=None, dx=32, dw=16, ld=64, lddh=64, yd=F32, hd=F32, dd=F32, wd=F32, ws=None, n=0):
        return L.tilec_rms_norm_backward(dy, h, rstd, None, dh, dx, dw, R, D, ld, ld, lddh, ld, yd, hd, dd, wd, ws, n, None)

    for kw in ({"yd": E4}, {"hd": E4}, {"wd": 9}, {"dh": 16, "dd": E5}):
        assert b(**kw) == TYPE, kw
    for kw in ({"R": -1}, {"D": 0}, {"dy": None}, {"h": None}, {"rstd": None}, {"dx": None}, {"ld": 63}, {"dh": 16, "lddh": 63},
               {"dx": 16}):  # dx in dy's place
        assert b(**kw) == VALUE, kw
    assert L.tilec_rms_norm_backward_workspace_bytes(1, 64, F32) == 0
    assert L.tilec_rms_norm_backward_workspace_bytes(3000, 64, F32) > 0
    assert L.tilec_rms_norm_backward_workspace_bytes(3000, 0, F32) == 0
    assert b(R=3000) == WORKSPACE


class Grad(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("n", ctypes.c_int64), ("dtype", ctypes.c_int32)]


def test_grad_norm_refusals():
    L = _lib.lib()

    def f(grads, norm=16, max_norm=1.0, ws=None, ws_bytes=0, counter=None, counter_bytes=0):
        return L.tilec_grad_norm((Grad * max(1, len(grads)))(*grads), len(grads), None, max_norm, norm, None, ws, ws_bytes,
                                 counter, counter_bytes, None)

    assert f([Grad(16, 4, E4)]) == TYPE
    for bad in ([Grad(None, 4, F32)], [Grad(16, -1, F32)]):
        assert f(bad) == VALUE
        assert L.tilec_scale_grads((Grad * 1)(*bad), 1, 16, None) == VALUE
    good = [Grad(16, 5000, F32), Grad(16, 0, BF16), Grad(None, 0, F32)]
    assert f(good, norm=None) == VALUE and f(good, max_norm=float("nan")) == VALUE
    assert L.tilec_grad_norm_workspace_bytes((Grad * 3)(*good), 3) == 16  # two chunks of 4096
    assert f(good) == WORKSPACE and f(good, ws=16, ws_bytes=16) == WORKSPACE and f(good, ws=16, ws_bytes=8, counter=16, counter_bytes=4) == WORKSPACE
    assert L.tilec_grad_norm(None, 2, None, 1.0, 16, None, None, 0, None, 0, None) == VALUE
    assert L.tilec_scale_grads((Grad * 3)(*good), 3, None, None) == VALUE
    # Large gradients: chunks of 64 Ki values at most.
    assert L.tilec_grad_norm_workspace_bytes((Grad * 1)(Grad(16, 1 << 30, BF16)), 1) == (1 << 30) // 65536 * 8


PROGRAM = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import tilec
x = torch.zeros(2, 300)
q = (x.to(torch.float8_e4m3fn), torch.ones(2, 3))
calls = [lambda: tilec.ext.rms_norm(x), lambda: tilec.ext.rms_norm_backward(x, x, x[:, 0]), lambda: tilec.ext.quantize_fp8(x),
         lambda: tilec.ext.dequantize_fp8(q), lambda: tilec.ext.linear_fp8(q, q), lambda: tilec.ext.grad_norm([x]),
         lambda: tilec.ext.clip_grads([x], 1.0)]
for call in calls:
    try:
        call()
    except TypeError:
        continue
    raise SystemExit("not refused")
"""


def test_torch_without_gpu_support():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_public_names():
    for name in ("rms_norm", "rms_norm_backward", "quantize_fp8", "dequantize_fp8", "linear_fp8", "grad_norm", "clip_grads"):
        assert name in tilec.ext.__all__ and callable(getattr(tilec.ext, name))


def test_wrong_arguments_raise():
    with pytest.raises(TypeError):
        tilec.ext.linear_fp8(1, 2)
    with pytest.raises(TypeError):
        tilec.ext.grad_norm(None)
    with pytest.raises(TypeError):
        tilec.ext.quantize_fp8("x")
    with pytest.raises(TypeError):
        tilec.ext.rms_norm([1.0])


def test_more_outputs_than_a_grid_has():
    most = (1 << 31) - 1024
    assert linear(M=most, N=most) == VALUE and "too many" in _lib.last_error()
    assert linear_bytes(most, 1, 16) == 0
