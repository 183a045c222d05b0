"""Build the CUDA library in-tree: heatvit_b200/_lib/libheatvit_b200.so.

One nvcc invocation per translation unit (parallel), linked into a shared
library with the CUDA runtime statically linked, for sm_100a only.  Beside it
_decode_native.so, the decode operators' calls from Python (a CPython module
on the installed torch's headers, linked against the library; left out where
there is no torch, which the library does not need).
"""

import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "_lib")
LIB = os.path.join(LIBDIR, "libheatvit_b200.so")
NATIVE = os.path.join(LIBDIR, "_decode_native.so")
NATIVE_SOURCE = os.path.join(CSRC, "hv_decode_torch.cpp")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr"]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps():
    files = sources() + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    files.append(os.path.join(os.path.dirname(HERE), "include", "heatvit_b200.h"))
    return files


def up_to_date():
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(f) <= t for f in _deps())


def native_made_for():
    """What the Python module is bound to beside its source: torch's version file and Python's ABI."""
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    with open(os.path.join(torch, "version.py")) as f:
        return sysconfig.get_config_var("EXT_SUFFIX") + "\n" + f.read()


def native_up_to_date():
    header = os.path.join(os.path.dirname(HERE), "include", "heatvit_b200.h")
    stamp = NATIVE + ".made_for"
    if not os.path.exists(NATIVE) or not os.path.exists(stamp):
        return False
    with open(stamp) as f:
        if f.read() != native_made_for():
            return False
    return all(os.path.getmtime(f) <= os.path.getmtime(NATIVE) for f in (NATIVE_SOURCE, header))


def build_native(force=False):
    """The decode operators' Python module, for the installed torch; None without one."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        print(f"heatvit_b200: torch is not installed, {os.path.basename(NATIVE)} (heatvit_b200.decode) is not built",
              file=sys.stderr)
        return None
    if not force and native_up_to_date():
        return NATIVE
    torch = spec.submodule_search_locations[0]
    cuda = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")
    tmp = NATIVE + ".tmp"
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared", "-Wall", NATIVE_SOURCE, "-o", tmp,
           "-isystem", os.path.join(torch, "include"),
           "-isystem", os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           "-isystem", cuda, "-I" + sysconfig.get_paths()["include"],
           "-L" + os.path.join(torch, "lib"), "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10",
           "-L" + LIBDIR, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{CXX} failed for {NATIVE_SOURCE}:\n{r.stderr}")
    os.replace(tmp, NATIVE)
    with open(NATIVE + ".made_for", "w") as f:
        f.write(native_made_for())
    return NATIVE


def build(force=False, verbose=False, ptxas_info=False):
    if not force and up_to_date():
        build_native()
        return LIB
    os.makedirs(os.path.join(LIBDIR, "obj"), exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas_info else []

    def compile_one(src):
        obj = os.path.join(LIBDIR, "obj", os.path.basename(src) + ".o")
        cmd = [NVCC, *ARCH, *FLAGS, *extra, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
        return obj, r.stderr

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, sources()))
    if verbose or ptxas_info:
        for _, err in results:
            if err:
                sys.stderr.write(err)
    objs = [o for o, _ in results]
    tmp = LIB + ".tmp"
    cmd = [NVCC, *ARCH, "-shared", "-o", tmp, *objs, "-Xcompiler", "-fPIC"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    build_native(force)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv)
    print(LIB)
