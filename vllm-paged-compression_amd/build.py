"""Builds libpaged_evict.so (all HIP kernels + the C ABI) for gfx950 and the host binding _host.so,
in-tree.

    python -m vllm_paged_compression_amd.build        (or)   python vllm-paged-compression_amd/build.py

hipcc cross-compiles without a GPU.  Objects go to build/ (git-ignored); the shared
library lands next to this file so that it travels with the source tree.
"""
import concurrent.futures
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libpaged_evict.so")
HOST_SRC = os.path.join(CSRC, "host_binding.cpp")
HOST = os.path.join(HERE, "_host.so")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
ARCH = "gfx950"
# -packed-fp32-ops: no packed 32-bit float instructions (v_pk_add/mul/fma_f32), which hipcc -O3
# otherwise forms from ordinary float code and some forms of which are not reliable on gfx950.  The
# host pass does not know the feature and says so once per file; that line is harmless.
FLAGS = ["--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
         "-Wno-unused-variable", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def host_binding_command():
    """g++ command of the host binding (csrc/host_binding.cpp): a CPython module over torch's C++
    tensors, linked with libpaged_evict.so next to it."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    tlib = os.path.join(os.path.dirname(torch.__file__), "lib")
    inc = [*include_paths(), sysconfig.get_paths()["include"], os.path.join(ROCM, "include")]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *("-isystem" + i for i in inc),
            HOST_SRC, "-o", HOST, "-L" + HERE, "-l:libpaged_evict.so", "-L" + tlib, "-ltorch_python", "-ltorch_cpu",
            "-lc10_hip", "-lc10", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + tlib]


def _headers_mtime():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    hs.append(os.path.join(os.path.dirname(HERE), "include", "paged_evict.h"))
    return max(os.path.getmtime(h) for h in hs)


def _compile(src, obj):
    subprocess.check_call(["hipcc", *FLAGS, "-c", src, "-o", obj])
    return obj


def build(force: bool = False, verbose: bool = True) -> str:
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    hm = _headers_mtime()
    jobs, objs = [], []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-4] + ".o")
        objs.append(obj)
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), hm):
            jobs.append((src, obj))
    if jobs:
        if verbose:
            print("hipcc:", ", ".join(os.path.basename(s) for s, _ in jobs), flush=True)
        with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            list(ex.map(lambda a: _compile(*a), jobs))
    if jobs or not os.path.exists(LIB):
        subprocess.check_call(["hipcc", "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", LIB, *objs])
        if verbose:
            print("linked", LIB, flush=True)
    if force or not os.path.exists(HOST) or os.path.getmtime(HOST) < max(os.path.getmtime(HOST_SRC), hm):
        if verbose:
            print("g++: host_binding.cpp", flush=True)
        subprocess.check_call(host_binding_command())
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
