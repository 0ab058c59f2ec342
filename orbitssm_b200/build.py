"""Build ``liborbit_b200.so`` in-tree with nvcc for sm_100a:  ``python -m orbitssm_b200.build``.

Each ``csrc/*.cu`` is compiled to an object file under ``csrc/_obj`` (in parallel, and only when it or a header is newer
than its object), then the objects are linked into the shared library next to this file.  ``csrc/host_calls.cpp`` (host code
against the headers of the installed torch, no kernels) becomes the extension module ``_orbit_host.so`` beside it; where it cannot be
built the library stands by itself, and the operators' Python host side serves every call."""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "_obj")
OUT = os.path.join(HERE, "liborbit_b200.so")
HOST_SRC, HOST_OUT = os.path.join(CSRC, "host_calls.cpp"), os.path.join(HERE, "_orbit_host.so")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        [os.path.join(os.path.dirname(HERE), "include", "orbit_b200.h")]


def _obj(src):
    return os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")


def _newer(path, deps):
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(d) > t for d in deps)


def stale() -> bool:
    return _newer(OUT, sources() + headers())


def host_tag() -> str:
    """What the host-call module is built against: its C++ ABI is the one of this torch and this Python alone."""
    import torch
    return f"orbit_host for torch {torch.__version__}, Python {sys.version_info.major}.{sys.version_info.minor};"


def host_matches() -> bool:
    """Does the built module carry the tag of the running torch and Python?"""
    with open(HOST_OUT, "rb") as f:
        return host_tag().encode() in f.read()


def build_host(force: bool = False) -> str:
    """The host-call extension (C++ against torch's headers; the torch libraries are found when the module is loaded)."""
    header = os.path.join(os.path.dirname(HERE), "include", "orbit_b200.h")
    if not force and not _newer(HOST_OUT, [HOST_SRC, header]) and host_matches():
        return HOST_OUT
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    nvcc = os.environ.get("NVCC", "nvcc")
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(nvcc) or "/usr/local/cuda/bin/nvcc")))
    inc = [sysconfig.get_paths()["include"], os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include")]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DORBIT_HOST_TAG="{host_tag()}"', *["-I" + i for i in inc],
           HOST_SRC, "-o", HOST_OUT, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("g++ failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
    return HOST_OUT


def build(force: bool = False, verbose: bool = False) -> str:
    if force or stale():
        build_library(force, verbose)
    try:
        build_host(force)
    except (RuntimeError, OSError, ImportError) as e:
        warnings.warn(f"the native host calls were not built, the Python host side of the operators serves every call: {e}", RuntimeWarning,
                      stacklevel=2)
    return OUT


def build_library(force: bool = False, verbose: bool = False) -> None:
    """The C-ABI library; needs nvcc alone."""
    nvcc = os.environ.get("NVCC", "nvcc")
    os.makedirs(OBJ, exist_ok=True)
    hdrs = headers()
    todo = [s for s in sources() if force or _newer(_obj(s), [s] + hdrs)]

    def compile_one(src):
        cmd = [nvcc, *FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-c", src, "-o", _obj(src)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        return src, cmd, res

    with ThreadPoolExecutor(max_workers=min(len(todo), os.cpu_count() or 1) or 1) as pool:
        for src, cmd, res in pool.map(compile_one, todo):
            if res.returncode != 0:
                raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
            if verbose:
                print(res.stderr)
    link = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", OUT, *[_obj(s) for s in sources()]]
    res = subprocess.run(link, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("link failed:\n" + " ".join(link) + "\n" + res.stdout + res.stderr)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
