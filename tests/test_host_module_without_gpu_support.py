"""tilec/_host.so as it is built against a torch without GPU support: from that torch's
headers and libraries alone, and it refuses tensors as ever."""

import os
import shutil
import subprocess
import sys

import pytest

from tilec import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import importlib.util, sys, torch
import tilec
from tilec import _lib
spec = importlib.util.spec_from_file_location("_host", sys.argv[1])
module = importlib.util.module_from_spec(spec)
spec.loader.exec_module(module)
_lib.host = lambda: module
x = torch.zeros(2, 300)
q = (x.to(torch.float8_e4m3fn), torch.ones(2, 3))
state = (torch.zeros(2, 300, dtype=torch.int8), torch.zeros(3))
e = tilec.ext
calls = [lambda: e.layer_norm(x), lambda: e.layer_norm_backward(x, x, x[:, 0], x[:, 0]),
         lambda: e.adamw_step([x], [x], [x], [x], step=1), lambda: e.adamw_values([state]), lambda: e.rms_norm(x),
         lambda: e.rms_norm_backward(x, x, x[:, 0]), lambda: e.quantize_fp8(x), lambda: e.dequantize_fp8(q),
         lambda: e.linear_fp8(q, q), lambda: e.grad_norm([x]), lambda: e.clip_grads([x], 1.0)]
for k, call in enumerate(calls):
    try:
        call()
    except TypeError:
        continue
    raise SystemExit(f"call {k} is not refused")
for call in (lambda: e.layer_norm(torch.zeros(2, 3, 4, 5)), lambda: e.grad_norm([])):
    try:
        call()
    except (TypeError, ValueError):
        continue
    raise SystemExit("not refused")
print("REFUSED")
"""


@pytest.fixture(scope="module")
def module(tmp_path_factory):
    where = tmp_path_factory.mktemp("host")
    out = str(where / "_host.so")
    r = subprocess.run(build.host_command(out, gpu=False), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    shutil.copy(build.LIB, where)  # it is looked for beside the module
    return out


def test_needs_no_gpu_library_of_torch(module):
    r = subprocess.run(["readelf", "-d", module], capture_output=True, text=True, check=True)
    needed = [line.split("[")[1].rstrip("]") for line in r.stdout.splitlines() if "(NEEDED)" in line]
    assert any("tilec_hip" in n for n in needed)
    assert not [n for n in needed if n.startswith(("libtorch_hip", "libc10_hip", "libtorch_cuda", "libc10_cuda", "libamdhip"))]
    r = subprocess.run(["nm", "-D", "-C", "--undefined-only", module], capture_output=True, text=True, check=True)
    assert not [line for line in r.stdout.splitlines() if "c10::hip" in line or "c10::cuda" in line or "empty_cuda" in line]


def test_needs_no_gpu_header_of_torch():
    cmd = build.host_command("unused", gpu=False)
    cmd = [c for c in cmd if c != "-shared"][:cmd.index("-o") - 1] + ["-M"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    headers = r.stdout.replace("\\\n", " ").split()
    assert any(h.endswith("torch/csrc/Dtype.h") for h in headers)
    assert not [h for h in headers if "/hip/" in h or "/cuda/" in h or "rocm" in h.split("dist-packages")[0]]


def test_refuses_tensors(module):
    r = subprocess.run([sys.executable, "-c", PROGRAM, module], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "REFUSED" in r.stdout, r.stdout + r.stderr
