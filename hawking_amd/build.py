"""Build the gfx950 HIP library (hawking_amd/lib/libhawking_hip.so) in-tree.

`python -m hawking_amd.build` compiles every source under hawking_amd/csrc
with hipcc for gfx950 and links one shared library exporting the C ABI of
include/hawking_hip.h.  Packed-FP32 instruction selection is disabled
(-packed-fp32-ops) for all device code, and MFMA accumulators live in
ordinary VGPRs (-amdgpu-mfma-vgpr-form).
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_obj")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libhawking_hip.so")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Werror",
    "-Wno-unused-command-line-argument",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA results in ordinary VGPRs: the epilogues read them directly instead
    # of copying each accumulator out of the AGPR file first
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    f"-I{os.path.join(ROOT, 'include')}",
]
SOURCES = ["hk_api.cpp", "hk_gemv2.hip", "hk_repack.hip", "hk_pack.hip", "hk_router.hip", "hk_moe.hip",
           "hk_moe_batch.hip", "hk_rice.hip", "hk_head.hip", "hk_container.cpp", "hk_parse.cpp", "hk_moe15.hip",
           "hk_moe_stack.hip", "hk_control.hip", "hk_rows_mixed.hip", "hk_rows_u3.hip", "hk_rows_q8.hip",
           "hk_rows_q4.hip", "hk_rows_bin.hip", "hk_rows.hip", "hk_group.hip", "hk_lora.hip", "hk_rows_api.cpp"]


def _compile(src: str) -> str:
    path = os.path.join(CSRC, src)
    obj = os.path.join(OBJ, os.path.splitext(src)[0] + ".o")
    lang = ["-x", "hip"] if src.endswith(".cpp") else []
    cmd = [HIPCC, *CFLAGS, *lang, "-c", path, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    jobs = min(len(SOURCES), int(os.environ.get("MAX_JOBS", "8")))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")
    return LIB


def build_oracle(verbose: bool = False) -> None:
    r = subprocess.run(["make", "-C", os.path.join(ROOT, "oracle")], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"oracle build failed:\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(r.stdout.strip())


if __name__ == "__main__":
    build_oracle(verbose=True)
    build(verbose=True)
    sys.exit(0)
