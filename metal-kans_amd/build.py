"""Build libkans_hip.so (gfx950) and, where torch is installed, its torch module in-tree.

    python metal-kans_amd/build.py [--jobs N] [--verbose]

Compiles every HIP translation unit under csrc/ with hipcc for gfx950 only and
links them into metal_kans/libkans_hip.so next to the Python package, so the
library travels with the source tree; csrc/kans_torch.cpp (host code) becomes
metal_kans/_kans_torch.so.  Packed-fp32 code generation is disabled
(``-target-feature -packed-fp32-ops``) for all device code.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "metal_kans")
LIB = os.path.join(OUT_DIR, "libkans_hip.so")
TORCH_LIB = os.path.join(OUT_DIR, "_kans_torch.so")
OBJ_DIR = os.path.join(HERE, "_build")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
HIPCC = os.environ.get("HIPCC", os.path.join(ROCM, "bin", "hipcc"))

DEVICE_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-ffp-contract=fast-honor-pragmas",
    # MFMA accumulators in VGPRs: the fused kernels keep <= 128 accumulator
    # registers per lane, and the AGPR form made the loop-carried accumulators
    # bounce between register files every step.
    "-mllvm", "--amdgpu-mfma-vgpr-form",
    "-Wno-unused-result",
]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def compile_one(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    cmd = [HIPCC, *DEVICE_FLAGS, "-I", CSRC, "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
    noise = [l for l in r.stderr.splitlines() if "packed-fp32-ops" not in l and l.strip()]
    if noise and verbose:
        print("\n".join(noise), file=sys.stderr)
    return obj


def build_torch_module(verbose: bool = False):
    """The autograd functions on torch tensors; None without torch."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    torch_dir = os.path.dirname(spec.origin)
    inc = os.path.join(torch_dir, "include")
    system = [inc, os.path.join(inc, "torch", "csrc", "api", "include"), os.path.join(ROCM, "include"),
              sysconfig.get_paths()["include"]]
    tmp = TORCH_LIB + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1",
           "-DUSE_ROCM=1", *(a for d in system for a in ("-isystem", d)), os.path.join(CSRC, "kans_torch.cpp"), "-o", tmp,
           "-L" + os.path.join(torch_dir, "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"the torch module does not build:\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


def build(jobs: int = 4, verbose: bool = False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=max(1, jobs)) as ex:
        torch_module = ex.submit(build_torch_module, verbose)
        objs = list(ex.map(lambda s: compile_one(s, verbose), srcs))
        torch_module.result()
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=min(8, os.cpu_count() or 1))
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.jobs, a.verbose))
