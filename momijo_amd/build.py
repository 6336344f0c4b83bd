"""Builds libmomijo_hip.so (the HIP kernels + the C ABI) in-tree for gfx950.

Each ``csrc/*.hip`` file is compiled to an object in ``momijo_amd/_build``
(in parallel) and the objects are linked into ``momijo_amd/libmomijo_hip.so``.
Run ``python -m momijo_amd.build`` or call :func:`build`.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD_DIR = os.path.join(HERE, "_build")
LIB_NAME = "libmomijo_hip.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
ARCH = "gfx950"

HIPCC = os.environ.get("HIPCC", shutil.which("hipcc") or "/opt/rocm/bin/hipcc")

# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 are generated (they are not
# trusted on the target machines).  The fp32 divide/sqrt flag keeps `a / b`
# the IEEE correctly rounded division, which the int8 quantizers rely on for
# bit-exact parity with a CPU fp32 division.
CFLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    # kernel arguments preloaded into SGPRs at wave launch (kernels with
    # scalar arguments: the GEMVs, quantizers, fp32 engine) instead of a
    # scalar load at the start of every wave; C3's GEMV 8.18 -> 8.15 us,
    # the W8A8 Linear 47.3 -> 46.8 us on MI355X
    "-mllvm", "-amdgpu-kernarg-preload-count=16",
    "-Wall",
    "-Wno-unused-function",
]
# Flags of single files.  gemm_f8.hip scales every result of the matrix cores on the
# vector unit: results in vector registers, not in accumulation registers that each
# have to be moved out first.
FILE_CFLAGS = {"gemm_f8.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"]}


def _compile(src: str) -> str:
    name = os.path.basename(src)
    obj = os.path.join(BUILD_DIR, name + ".o")
    cmd = [HIPCC, *CFLAGS, *FILE_CFLAGS.get(name, []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}")
    return obj


def build(verbose: bool = False) -> str:
    """Compile every kernel source and link the shared library; returns its path."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    if not srcs:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = min(len(srcs), max(1, (os.cpu_count() or 4)), 8)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = LIB_PATH + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}")
    os.replace(tmp, LIB_PATH)
    if verbose:
        print(f"built {LIB_PATH} from {len(srcs)} sources", flush=True)
    return LIB_PATH


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
