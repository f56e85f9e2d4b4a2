"""Build libaspidagpu.so (the HIP C-ABI library) in-tree for gfx950.

    python -m aspida_amd.build          # or: python aspida_amd/build.py

Compiles every .hip file under aspida_amd/csrc/ with hipcc into one shared
library next to this file.  Each translation unit is compiled in parallel,
then linked.
"""
import concurrent.futures
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libaspidagpu.so")
OBJ_DIR = os.path.join(HERE, "_build")
ARCH = os.environ.get("ASPIDA_OFFLOAD_ARCH", "gfx950")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall",
    # No packed-FP32 VALU instructions anywhere in the device code.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I", os.path.join(HERE, "..", "include"),
]


# Per-source flags.  kq_mv_mfma.hip (the batch-1 matrix-core kernels): MFMA
# results in VGPRs rather than AGPRs, which drops a v_accvgpr_read per result
# from the 64-row column loops (Q2_K / Q3_K / Q5_K launches of 28672x4096 and
# up 2-7% faster, the 8B decode +0.2%); the small-batch sources measured equal
# or slower with it (Q4_K 4096^2 at 64 vectors +12%), so only this file.
# kv4_attn.hip, kv4_weigh.hip, kv4_prefill.hip: without it the sums sit in
# AGPRs, and every product with a vector instruction moves them (decode
# attention with heads of 128: 228 registers, 196 with it).
EXTRA_FLAGS = {"kq_mv_mfma.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
               "kv4_attn.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
               "kv4_weigh.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
               "kv4_prefill.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]}


def _compile(src):
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    cmd = [HIPCC, *CFLAGS, *EXTRA_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass does not know the device feature flag; drop that note.
    err = "\n".join(l for l in r.stderr.splitlines() if "packed-fp32-ops" not in l)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{err}")
    if err.strip():
        sys.stderr.write(err + "\n")
    return obj


def build(verbose=True):
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = OUT + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, OUT)
    if verbose:
        print(f"built {OUT}")
    return OUT


if __name__ == "__main__":
    build()
