"""Build libatlasinfer_amd.so (the gfx950 kernels and their C ABI) in-tree.

    python -m atlasinfer_amd.build

Each .hip file under csrc/ is compiled for gfx950 in parallel and the objects
are linked into atlasinfer_amd/libatlasinfer_amd.so, which the host side loads
with ctypes.
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
OUT = os.path.join(HERE, "libatlasinfer_amd.so")
OBJ_DIR = os.path.join(HERE, "_build")

ARCH = "gfx950"
HIPCC = os.environ.get("HIPCC", shutil.which("hipcc") or "/opt/rocm/bin/hipcc")
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # every floating-point operation rounds as written; fused multiply-adds
    # appear only where the source asks for them
    "-ffp-contract=off",
    # no packed-f32 arithmetic in generated code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
]


# per-file additions: the quantized-linear and attention kernels keep MFMA
# accumulators in ordinary VGPRs (the accumulator-register form made the
# compiler shuffle accumulators between register files inside the K loop)
FILE_FLAGS = {f: ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]
              for f in ("aq_qlinear.hip", "aq_qlinear_mid.hip", "aq_kv4.hip", "aq_window.hip", "aq_paged_attention.hip")}


def _compile(src: str) -> str:
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    cmd = [HIPCC, *FLAGS, *FILE_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
    return obj


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = OUT + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, OUT)
    if verbose:
        print(f"built {OUT}")
    return OUT


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
