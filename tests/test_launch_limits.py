"""Grids of the calls with the most rows, columns or nothing at all, on the host: the
library is loaded beside a small one whose hipLaunchKernel writes the launches down
instead of enqueueing them, so no memory of these sizes and no GPU is needed.  A grid
has fewer than 2^32 threads along an axis, and at most 2^16 workgroups along y and z."""

import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RECORDER = r"""
#include <cstddef>
struct Dim3 { unsigned x, y, z; };
static unsigned kept[6 * 1024];
static int count;
extern "C" {
int hipLaunchKernel(const void*, Dim3 grid, Dim3 block, void**, size_t, void*) {
  const unsigned all[6] = {grid.x, grid.y, grid.z, block.x, block.y, block.z};
  for (int i = 0; count < 1024 && i < 6; ++i) kept[6 * count + i] = all[i];
  ++count;
  return 0;
}
int hipGetLastError() { return 0; }
// What kernel<<<...>>> keeps between its configuration and hipLaunchKernel.
static Dim3 grid_of, block_of;
int __hipPushCallConfiguration(Dim3 grid, Dim3 block, size_t, void*) {
  grid_of = grid, block_of = block;
  return 0;
}
int __hipPopCallConfiguration(Dim3* grid, Dim3* block, size_t* shared, void** stream) {
  *grid = grid_of, *block = block_of, *shared = 0, *stream = nullptr;
  return 0;
}
int recorded(unsigned* out) {
  const int n = count;
  for (int i = 0; i < 6 * n && i < 6 * 1024; ++i) out[i] = kept[i];
  count = 0;
  return n;
}
}
"""

# (The package itself would load torch, and with it the runtime's library first.)
PROGRAM = """
import ctypes, importlib.util, json, sys
recorder = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
spec = importlib.util.spec_from_file_location("binding", sys.argv[2])
binding = importlib.util.module_from_spec(spec)
spec.loader.exec_module(binding)
L = binding.lib()
out = (ctypes.c_uint32 * (6 * 1024))()
answers = []
for name, args in json.load(sys.stdin):
    rc = getattr(L, name)(*args)
    n = recorder.recorded(out)
    answers.append([rc, [list(out[6 * i:6 * i + 6]) for i in range(n)]])
print("ANSWERS" + json.dumps(answers))
"""

F32, BF16, E4 = 0, 1, 2
AT, ROOM = 1 << 20, 1 << 60  # an address, and room for anything: nothing reads or writes there
MOST = (1 << 31) - 1024
TINY = 1e-5


def linear(M, N, K, od, x=AT, w=AT, ldx=None, ldw=None):
    return ("tilec_linear_fp8", [x, AT, w, AT, AT, M, N, K, K if ldx is None else ldx, K if ldw is None else ldw, N, 1, 1, 1, 1,
                                 E4, E4, od, 1, 1, AT, ROOM, AT, ROOM, None])


CASES = {}
for _od in (F32, BF16):
    for _M, _N in ((100, 100), (1 << 30, 4), ((1 << 30) + 5, 64), (1, MOST), (16, 1 << 30), (MOST, 1)):
        CASES[f"no features {_M} x {_N} {_od}"] = linear(_M, _N, 0, _od)
for _od in (F32, BF16):
    # Operands that are copied first: a stride, or an address, off 16 bytes.
    CASES[f"copied x {_od}"] = linear((1 << 30) + 1000, 1, 33, _od)
    CASES[f"copied x, short rows {_od}"] = linear(MOST, 1, 16, _od, x=AT + 1)
    CASES[f"copied weight {_od}"] = linear(4, (1 << 30) + 1000, 64, _od, w=AT + 8)
    CASES[f"copied weight, {(1 << 22) - 3} features {_od}"] = linear(16, 60000, (1 << 22) - 3, _od)
    CASES[f"both copied {_od}"] = linear(1 << 30, 1 << 5, 40, _od)


def rms_backward(R, D, hd, dw=AT):
    return ("tilec_rms_norm_backward", [AT, 2 * AT, AT, None, None, 3 * AT, dw, R, D, D, D, D, D, hd, hd, hd, F32, AT, ROOM, None])


for _hd in (F32, BF16):
    for _R, _D in ((0, 1), (0, 1 << 26), (0, MOST), (1, MOST), (3, 1 << 29), (MOST, 1), (1 << 24, 64), (1 << 20, 4096), (1 << 15, 1 << 17)):
        CASES[f"RMS norm backward {_R} x {_D} {_hd}"] = rms_backward(_R, _D, _hd)


def layer_norm_backward(R, D, xd, dw=AT, db=2 * AT):
    return ("tilec_layer_norm_backward", [AT, AT, AT, AT, None, AT, dw, db, R, D, D, D, D, xd, xd, F32, AT, ROOM, None])


for _xd in (F32, BF16):
    for _R, _D in ((0, 1), (0, 1 << 25), (0, MOST), (1, MOST), (3, 1 << 29), (MOST, 1), (1 << 24, 64), (1 << 20, 4096), (1 << 15, 1 << 17)):
        CASES[f"layer norm backward {_R} x {_D} {_xd}"] = layer_norm_backward(_R, _D, _xd)
    CASES[f"layer norm backward, no weight {_xd}"] = layer_norm_backward(0, 1 << 26, _xd, dw=None)
    CASES[f"layer norm backward, no bias {_xd}"] = layer_norm_backward(0, 1 << 26, _xd, db=None)

# The other entry points at their longest and widest.
LARGE = [(1, MOST), (MOST, 1), (128, 1 << 30), (1 << 30, 128), (1 << 24, 8192), (1 << 15, 1 << 22), ((1 << 26) + 1, 2049)]
for _t in (F32, BF16):
    for _R, _D in LARGE:
        CASES[f"RMS norm {_R} x {_D} {_t}"] = ("tilec_rms_norm", [AT, None, None, AT, None, None, AT, _R, _D, _D, 0, _D, 0, 0, 0, _t,
                                               F32, _t, F32, TINY, None])
        CASES[f"RMS norm to 8 bits {_R} x {_D} {_t}"] = ("tilec_rms_norm", [
            AT, AT, None, AT, AT, AT, AT, _R, _D, _D, _D, -(-_D // 16) * 16, _D, 1, 1, _t, F32, E4, F32, TINY, None])
        CASES[f"layer norm {_R} x {_D} {_t}"] = ("tilec_layer_norm", [AT, None, None, AT, AT, AT, _R, _D, _D, _D, _t, _t, F32, TINY,
                                                 None])
        for _block in (1, 128):
            for _trans in (0, 1):
                CASES[f"quantise {_R} x {_D} {_t} {_block} {_trans}"] = ("tilec_quantize_fp8", [
                    AT, AT, AT, _R, _D, _R if _trans else _D, -(-_D // 16) * 16, 1, 1, _trans, _t, E4, _block, None])
            CASES[f"values {_R} x {_D} {_t} {_block}"] = ("tilec_dequantize_fp8", [AT, AT, AT, _R, _D, _D, _D, 1, 1, E4, _t, _block,
                                                          None])
    for _M, _N, _K in ((1, MOST, 16), (16, 1 << 30, 130), (MOST, 1, 16), (1 << 30, 64, 128), (1 << 20, 1 << 17, 256),
                       (1 << 17, 1 << 20, 256), (8192, 8192, 1 << 22)):
        CASES[f"product {_M} x {_N} x {_K} {_t}"] = linear(_M, _N, _K, _t)


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    where = tmp_path_factory.mktemp("recorder")
    src, lib = where / "recorder.cpp", where / "recorder.so"
    src.write_text(RECORDER)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", str(src), "-o", str(lib)], check=True, timeout=120)
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(lib), os.path.join(ROOT, "tilec", "_lib.py")], cwd=ROOT,
                       input=json.dumps(list(CASES.values())), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    text = r.stdout[r.stdout.index("ANSWERS") + len("ANSWERS"):]
    return dict(zip(CASES, json.loads(text)))


@pytest.mark.parametrize("name", CASES)
def test_grids(name, answers):
    rc, launches = answers[name]
    assert rc == 0 and launches
    for gx, gy, gz, bx, by, bz in launches:
        assert 0 < bx * by * bz <= 1024
        assert 0 < gx * bx < 1 << 32 and 0 < gy <= 1 << 16 and 0 < gz <= 1 << 16, (gx, gy, gz, bx)
