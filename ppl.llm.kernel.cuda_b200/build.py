"""Builds the sm_100a shared library in-tree, lib/libpplb200_i8i8.so, and (where torch is installed, whose tensors it reads) the
compiled part of the Python binding, lib/pplb200_attention_binding.<python>.torch-<version>.so: another torch or Python needs another.
For tests, lib/libpplb200_impatient_prefix.so is built beside them.

    python build.py [--force] [--verbose]

nvcc cross-compiles without a GPU.  The explicit -gencode form matters: tcgen05 is only
accepted for the arch-specific target sm_100a, and plain -arch=sm_100a would also emit a
generic compute_100 PTX image in which it is rejected.
"""
import concurrent.futures
import importlib.util
import os
import runpy
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libpplb200_i8i8.so")
SOURCES = ["capi.cu", "quantize.cu", "rmsnorm_quantize.cu", "activation_requant.cu", "gemm_i8_tcgen05.cu", "gemm_i8_decode.cu", "gemm_i8_token_pair.cu", "tensor_parallel.cu", "p2p_row_parallel.cu", "no_alloc.cu", "rotary_kv.cu", "paged_attention.cu", "paged_attention_general.cu", "shared_prefix.cu", "block_sparse.cu", "probes.cu"]
# For tests alone: the library with a kernel for shared prefixes in which the warp that issues the products has no patience for the last two tasks' values.
TEST_LIB = os.path.join(LIBDIR, "libpplb200_impatient_prefix.so")
TEST_FLAGS = ["-DPPLB200_IMPATIENT_PREFIX"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
BINDING_SOURCE = os.path.join(CSRC, "attention_binding.cpp")
FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def torch_home():
    """Where torch is installed, or None.  It is not imported: that takes longer than a build with nothing to do."""
    spec = importlib.util.find_spec("torch")
    return spec.submodule_search_locations[0] if spec is not None else None


def torch_version():
    return runpy.run_path(os.path.join(torch_home(), "version.py"))["__version__"]


def binding_path():
    """As pplb200/attention.py looks for it."""
    return os.path.join(LIBDIR, "pplb200_attention_binding.%s.torch-%s.so" % (sys.implementation.cache_tag, torch_version()))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False):
    os.makedirs(LIBDIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers += [os.path.join(HERE, "..", "include", f) for f in ("pplb200_i8i8.h", "pplb200_attention.h")]
    objs, cmds = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(LIBDIR, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + headers):
            cmds.append([NVCC] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o])
            if verbose:
                print(" ".join(cmds[-1]))
    impatient, prefix = os.path.join(LIBDIR, "shared_prefix_impatient.o"), os.path.join(CSRC, "shared_prefix.cu")
    if force or _stale(impatient, [prefix] + headers):
        cmds.append([NVCC] + FLAGS + TEST_FLAGS + ["-c", prefix, "-o", impatient])
    with concurrent.futures.ThreadPoolExecutor(os.cpu_count()) as pool:  # files compile side by side
        list(pool.map(lambda cmd: subprocess.run(cmd, check=True), cmds))
    if force or _stale(LIB, objs):
        cmd = [NVCC, "-shared", "-o", LIB] + objs + ["-ldl"]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    parts = [impatient if os.path.basename(o) == "shared_prefix.o" else o for o in objs]
    if force or _stale(TEST_LIB, parts):
        subprocess.run([NVCC, "-shared", "-o", TEST_LIB] + parts + ["-ldl"], check=True)
    home = torch_home()
    if home is None:
        print("torch is not installed: the compiled part of the Python binding (rotary positions, cache, attention) is not built")
    elif force or _stale(binding_path(), [BINDING_SOURCE] + headers):
        cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-fvisibility=hidden", "-I" + sysconfig.get_paths()["include"],
               "-isystem", os.path.join(home, "include"), "-isystem", os.path.join(home, "include", "torch", "csrc", "api", "include"),
               BINDING_SOURCE, "-o", binding_path(), "-L" + os.path.join(home, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
