"""Build libsplat_hip.so from ../csrc with hipcc for gfx950 (cross-compiles without a GPU).

Objects go to ../_build/, the library next to this file so it ships with the package tree.
"""

from __future__ import annotations

import os
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(ROOT, "csrc")
OBJ_DIR = os.path.join(ROOT, "_build")
LIB_NAME = "libsplat_hip.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
ARCH = os.environ.get("SPLAT_HIP_ARCH", "gfx950")

# Packed fp32 VALU forms are disabled for all device code; atomics on coarse-grained memory use the
# hardware fp32 add.
HIP_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-munsafe-fp-atomics",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]
# Per-source extra flags: the binning must round every fp32 op separately (no FMA contraction); matrix instructions of
# the products and the attention keep their accumulators in vector registers (in accumulation registers the compiler moves
# them to vector registers and back around every softmax step).
_VGPR_ACC = ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]
SOURCES = {
    "capi.hip": [],
    "bin.hip": ["-ffp-contract=off"],
    "render.hip": [],
    "norm.hip": [],
    "linear.hip": _VGPR_ACC,
    "attend.hip": _VGPR_ACC,
    "rotary.hip": [],
    "token_norm.hip": [],
    "paged.hip": _VGPR_ACC,
}


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    return os.path.join(rocm, "bin", "hipcc")


def build(verbose: bool = False) -> str:
    """Compile every source (in parallel) and link the shared library. Returns the library path."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    procs = []
    objs = []
    for src, extra in SOURCES.items():
        obj = os.path.join(OBJ_DIR, src.replace(".hip", ".o"))
        objs.append(obj)
        cmd = [hipcc(), *HIP_FLAGS, *extra, "-I", CSRC, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(f"--- {src}\n{out}")
        elif verbose and out.strip():
            print(out, flush=True)
    if failed:
        raise RuntimeError("hipcc failed:\n" + "\n".join(failed))
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
