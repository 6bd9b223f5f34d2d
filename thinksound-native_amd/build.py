"""Build libtsn.so (gfx950) in-tree with hipcc: thinksound-native_amd/lib/libtsn.so.

Every source is compiled for gfx950 only, with packed-FP32 instruction selection disabled
(-Xclang -target-feature -Xclang -packed-fp32-ops), objects in parallel, then linked -shared.
"""
import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "lib")
OBJ_DIR = os.path.join(HERE, "_build")
LIB = os.path.join(OUT_DIR, "libtsn.so")

SOURCES = ["gemm.hip", "attention.hip", "ops.hip", "vae.hip", "enc.hip", "netops.hip", "blockops.hip", "diffattn.hip", "noalloc.hip", "runtime.cpp", "graph.cpp", "gguf.cpp", "dit.cpp", "refdit.cpp", "refcond.cpp", "vae.cpp", "encoders.cpp", "tokenizers.cpp", "synth.cpp", "capi.cpp"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
COMMON = ["-std=c++17", "-O3", "-fPIC", "-Wall", "-Wno-unused-function",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


# attention.hip produces no NaN (every key block holds a valid key, masked scores are -inf): with
# NaNs ruled out the compiler drops the quieting max before each max of the softmax
EXTRA = {"attention.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"],
         # products stay in VGPRs, where the softmax reads and rescales them (the kernel for few rows has a SIMD's
         # whole register file a wave and would get AGPRs, and two moves for every value)
         "diffattn.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]}


def _compile(src):
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    cmd = ([HIPCC, "--offload-arch=" + ARCH] + COMMON + EXTRA.get(src, []) +
           ["-x", "hip", "-c", os.path.join(CSRC, src), "-o", obj])
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("compile failed: %s\n%s\n%s" % (" ".join(cmd), r.stdout, r.stderr))
    return obj


def build(verbose=False):
    os.makedirs(OUT_DIR, exist_ok=True)
    os.makedirs(OBJ_DIR, exist_ok=True)
    workers = min(len(SOURCES), max(1, min(os.cpu_count() or 1, 8)))
    with cf.ThreadPoolExecutor(workers) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=" + ARCH, "-shared", "-fPIC", "-Wl,--no-undefined", "-o", tmp] + objs + ["-lpthread"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed: %s\n%s\n%s" % (" ".join(cmd), r.stdout, r.stderr))
    os.replace(tmp, LIB)
    if verbose:
        print("built", LIB)
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
