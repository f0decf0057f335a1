"""Build libtilec_hip.so in-tree with hipcc for gfx950.

    python -m tilec.build            # compile + link (always rebuilds)

Each .hip file under csrc/ is compiled to an object in csrc/_build/ in
parallel, then linked into tilec/libtilec_hip.so, which ext.py loads with
ctypes.  The library is written for MI355X only (--offload-arch=gfx950).
csrc/host.cpp, host code that reads torch tensors, becomes the Python module
tilec/_host.so beside it.
"""

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJDIR = os.path.join(CSRC, "_build")
LIB = os.path.join(HERE, "libtilec_hip.so")
HOST = os.path.join(HERE, "_host.so")
ARCH = "gfx950"

# -packed-fp32-ops: keep v_pk_{add,mul,fma}_f32 out of the generated code.
CFLAGS = [
    "-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-unused-command-line-argument",
]


def hipcc():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm is required to build libtilec_hip.so)")


def _compile(src):
    obj = os.path.join(OBJDIR, os.path.basename(src).replace(".hip", ".o"))
    cmd = [hipcc(), *CFLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def _host():
    """tilec/_host.so: a CPython module against torch's headers and libraries and
    libtilec_hip.so beside it."""
    import torch
    from torch.utils import cpp_extension
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = HOST + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I" + sysconfig.get_paths()["include"], *("-isystem" + p for p in cpp_extension.include_paths()),
           os.path.join(CSRC, "host.cpp"), "-o", tmp, "-L" + torch_lib, "-Wl,-rpath," + torch_lib,
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-L" + HERE, "-Wl,-rpath,$ORIGIN", "-ltilec_hip"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building {HOST} failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, HOST)


def build(verbose=False):
    os.makedirs(OBJDIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = LIB + ".tmp"
    # --no-undefined: a kernel whose host stub the compiler dropped fails here,
    # not when the library is first loaded.
    cmd = [hipcc(), "-shared", "-fPIC", f"--offload-arch={ARCH}", "-Wl,--no-undefined", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    _host()
    if verbose:
        print(f"built {LIB} and {HOST}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
