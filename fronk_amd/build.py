"""Build the MI355X libraries in-tree (no JIT cache, no site-packages).

libfronk_hip.so      HIP kernels + C ABI (include/fronk_hip.h), gfx950 only.
_dense.so            fronk_amd.dense's side of it over torch tensors
                     (host/dense_module.cpp).
libfr_hip.so         the "hip" fr_backend vtable (host/hip.c, plain C11),
                     compiled against the reference's own src/ headers where
                     they lie (hidden size fixed there at 2560) and linked
                     against libfronk_hip.so. Its remaining symbols (hw_probe,
                     fr_vectors_check, ...) come from the reference program it
                     is loaded into. Built only when the reference is present.
"""
import os
import subprocess
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
# The expert engine (fronk_hip.hip within engine.hip), and the dense operators around it.
HIP_SRCS = [os.path.join(HERE, "csrc", n) for n in ("engine.hip", "delta.hip", "q4.hip", "kv.hip")]
HIP_LIB = os.path.join(HERE, "libfronk_hip.so")
VTABLE_SRC = os.path.join(HERE, "host", "hip.c")
VTABLE_LIB = os.path.join(HERE, "libfr_hip.so")
DENSE_SRC = os.path.join(HERE, "host", "dense_module.cpp")
DENSE_LIB = os.path.join(HERE, "_dense.so")
REFERENCE_SRC = os.path.join(os.environ.get("FRONK_REFERENCE", "/root/reference"), "src")

# Packed-FP32 instructions are disabled for every HIP translation unit.
HIPCC_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
               "-I" + os.path.join(ROOT, "include")]


def build_hip(verbose=False):
    """One object per source, compiled side by side, and one library of them."""
    def compile_one(src):
        obj = src + ".o"
        subprocess.run(["hipcc", *HIPCC_FLAGS, "-c", src, "-o", obj], check=True, capture_output=not verbose)
        return obj
    with ThreadPoolExecutor(len(HIP_SRCS)) as pool:
        objs = list(pool.map(compile_one, HIP_SRCS))
    subprocess.run(["hipcc", "--offload-arch=gfx950", "-shared", *objs, "-o", HIP_LIB + ".tmp"], check=True,
                   capture_output=not verbose)
    for obj in objs:
        os.remove(obj)
    os.replace(HIP_LIB + ".tmp", HIP_LIB)
    return HIP_LIB


def build_vtable(verbose=False):
    cmd = ["gcc", "-std=c11", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror",
           "-D_POSIX_C_SOURCE=200809L", "-D_DEFAULT_SOURCE", "-DFR_BENCH_RUNTIME=1", "-DFR_HIP_MODULE=1", "-I" + REFERENCE_SRC, "-I" + os.path.join(ROOT, "include"),
           VTABLE_SRC, "-o", VTABLE_LIB + ".tmp", "-L" + HERE, "-lfronk_hip", "-Wl,-rpath,$ORIGIN", "-lm"]
    subprocess.run(cmd, check=True, capture_output=not verbose)
    os.replace(VTABLE_LIB + ".tmp", VTABLE_LIB)
    return VTABLE_LIB


def build_dense(verbose=False):
    """The torch side of the dense operators, linked to libfronk_hip.so."""
    import torch
    at = os.path.dirname(torch.__file__)
    include = [os.path.join(ROOT, "include"), os.path.join(at, "include"),
               os.path.join(at, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"]]
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", *("-I" + i for i in include),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", DENSE_SRC, "-o", DENSE_LIB + ".tmp",
           "-L" + HERE, "-lfronk_hip", "-Wl,-rpath,$ORIGIN", "-L" + os.path.join(at, "lib"), "-ltorch_python",
           "-ltorch_cpu", "-lc10"]
    subprocess.run(cmd, check=True, capture_output=not verbose)
    os.replace(DENSE_LIB + ".tmp", DENSE_LIB)
    return DENSE_LIB


def build_all(verbose=False):
    build_hip(verbose)
    build_dense(verbose)
    if os.path.isdir(REFERENCE_SRC):
        build_vtable(verbose)


if __name__ == "__main__":
    build_all(verbose=True)
