"""Ahead-of-time build of libfxb200.so (sm_100a) from csrc/*.cu.

The reference compiles its HIP sources at run time with hiprtc
(ml/fxgpu/hip_kernel.py:50-131); this build compiles every CUDA source once,
in parallel, with nvcc for sm_100a and links one shared library with a plain C
ABI (include/fxb200.h). cudart is linked statically and the driver API is
reached through cudaGetDriverEntryPoint, so the library loads on a machine
without libcuda (symbol checks on CPU) and runs wherever the driver is present.

    python -m fxb200.build          # from radeon-igpu-forge_b200/
"""
import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(PKG_ROOT, "csrc")
LIB_DIR = os.path.join(PKG_ROOT, "lib")
OBJ_DIR = os.path.join(LIB_DIR, "obj")
LIB_PATH = os.path.join(LIB_DIR, "libfxb200.so")
REPO_ROOT = os.path.dirname(PKG_ROOT)
INCLUDE = os.path.join(REPO_ROOT, "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
         "--expt-relaxed-constexpr", "-I" + INCLUDE, "-I" + CSRC]


def _nvcc():
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found (CUDA toolkit required to build libfxb200)")
    return exe


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers_mtime():
    ts = [os.path.getmtime(os.path.join(CSRC, f)) for f in os.listdir(CSRC)
          if f.endswith((".cuh", ".h"))]
    ts.append(os.path.getmtime(os.path.join(INCLUDE, "fxb200.h")))
    return max(ts)


def _compile(src, verbose=False):
    obj = os.path.join(OBJ_DIR, src[:-3] + ".o")
    cmd = [_nvcc()] + ARCH + FLAGS + ["-c", os.path.join(CSRC, src), "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj, r.stderr


def _binding_key():
    """What lib/_fxbind.so depends on besides its sources: the versions of torch and Python; None without torch."""
    if importlib.util.find_spec("torch") is None:
        return None
    return f"torch {importlib.metadata.version('torch')}, Python {sys.version}"


def _build_binding(force=False):
    """lib/_fxbind.so from csrc/bind.cpp, against torch's headers (host code).
    Only the generation operators need it: without torch it is left out."""
    src, out = os.path.join(CSRC, "bind.cpp"), os.path.join(LIB_DIR, "_fxbind.so")
    key, stamp = _binding_key(), out + ".key"
    if key is None:
        sys.stderr.write("torch is not installed: libfxb200.so is built, _fxbind.so (generation over a KV cache) not\n")
        return
    built_for = None
    if os.path.exists(out) and os.path.exists(stamp):
        with open(stamp) as f:
            built_for = f.read()
    newest = max(os.path.getmtime(src), os.path.getmtime(os.path.join(INCLUDE, "fxb200.h")))
    if not force and built_for == key and os.path.getmtime(out) >= newest:
        return
    import torch
    home = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")
    headers = os.path.join(home, "include")
    paths = [INCLUDE, headers, os.path.join(headers, "torch", "csrc", "api", "include"), cuda,
             sysconfig.get_path("include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *("-I" + p for p in paths), src, "-o", out + ".tmp", "-L" + os.path.join(home, "lib"),
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for bind.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(out + ".tmp", out)
    with open(stamp, "w") as f:
        f.write(key)


def build(force=False, verbose=False, jobs=None):
    """Compile stale objects and relink; returns the library path."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    hdr = _headers_mtime()
    todo, objs = [], []
    for src in _sources():
        obj = os.path.join(OBJ_DIR, src[:-3] + ".o")
        objs.append(obj)
        stale = (force or not os.path.exists(obj)
                 or os.path.getmtime(obj) < max(hdr, os.path.getmtime(os.path.join(CSRC, src))))
        if stale:
            todo.append(src)
    if todo:
        n = jobs or min(len(todo), os.cpu_count() or 4)
        with cf.ThreadPoolExecutor(max_workers=n) as ex:
            for obj, log in ex.map(lambda s: _compile(s, verbose), todo):
                if verbose and log:
                    sys.stderr.write(log)
    if todo or not os.path.exists(LIB_PATH):
        tmp = LIB_PATH + ".tmp"
        cmd = [_nvcc()] + ARCH + ["-shared", "-cudart", "static", "-o", tmp] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB_PATH)
    _build_binding(force)
    return LIB_PATH


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(p)
