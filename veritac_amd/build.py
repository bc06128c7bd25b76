"""Build recipe for libvt_hip_gemm.so (gfx950) -- run at build time only.

    python -m veritac_amd.build          # compile veritac_amd/libvt_hip_gemm.so

hipcc cross-compiles for gfx950 without a GPU. The library is built in-tree
so it travels with the source tree; nothing builds at import time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
SOURCES = [os.path.join(PKG_DIR, "csrc", "vt_hip_gemm.hip")]
# device and host code that SOURCES include
PARTS = [os.path.join(PKG_DIR, "csrc", name) for name in ("vt_scaled.h", "vt_norm.h", "vt_loss.h", "vt_adapter.h")]
INCLUDE = os.path.join(ROOT, "include")
LIB_PATH = os.path.join(PKG_DIR, "libvt_hip_gemm.so")
ARCH = "gfx950"

# -packed-fp32-ops is disabled for every HIP translation unit (the host pass
# warns that it does not know the feature; that is harmless).
HIPCC_FLAGS = [
    "--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-shared",
    "-Wall", "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]
# hipRTC compiles the emitted loop-nest kernels at run time.
LINK_FLAGS = ["-L/opt/rocm/lib", "-lhiprtc", "-Wl,-rpath,/opt/rocm/lib"]


def hipcc():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def build(verbose=False):
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc()] + HIPCC_FLAGS + ["-I", INCLUDE] + SOURCES + LINK_FLAGS + ["-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in proc.stderr.splitlines() if noise not in l)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed (%d):\n%s" % (proc.returncode, err))
    if verbose and err.strip():
        print(err, file=sys.stderr)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
