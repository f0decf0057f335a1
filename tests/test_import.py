"""The package on a torch built without GPU support: it imports, its host-side
helpers work, and calls refuse CPU tensors."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import tilec
assert tilec.ext.plan(100) == (256, 1) and tilec.ext.mm_configs(4, 64, 4)
x = torch.zeros(2, 3)
calls = [lambda: tilec.ext.linear_cross_entropy(x, x, torch.zeros(2, dtype=torch.int64)),
         lambda: tilec.ext.layer_norm(x), lambda: tilec.ext.layer_norm_backward(x, x, x[:, 0], x[:, 0]),
         lambda: tilec.ext.adamw_step([x], [x], [x], [x], step=1), lambda: tilec.ext.matrix_mul(x, x.t()),
         lambda: tilec.ext.sum(x)]
for call in calls:
    try:
        call()
    except TypeError:
        continue
    raise SystemExit("not refused")
"""


def test_torch_without_gpu_support():
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
