"""Builds libbmo.so in-tree (bmo_jetson_b200/lib/libbmo.so) for sm_100a.

CUDA sources are compiled by nvcc with ``-gencode arch=compute_100a,code=sm_100a``,
host sources by g++; the shared library links the CUDA runtime statically so it
does not depend on whichever libcudart a host process already loaded.
Rebuilds only objects whose source or headers changed.  Where torch with CUDA
and Python's headers are installed, the torch binding of the paged cache is
built beside it (bmo_jetson_b200/lib/_paged.<tag>.so, the tag made of torch's and
Python's versions and of the sources).

    python -m bmo_jetson_b200.build [--force] [-j N]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import hashlib
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "lib", "obj")
LIB = os.path.join(HERE, "lib", "libbmo.so")
# torch binding of the paged cache (bmo_jetson_b200/paged.py): an extension module, built where torch is installed
BINDING_SRC = os.path.join(HERE, "binding", "paged_torch.cpp")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = "/usr/bin/g++"
CUDA_INC = "/usr/local/cuda/include"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]

NVCC_FLAGS = ARCH + ["-O3", "-std=c++17", "-lineinfo", "-ccbin", CXX, "-Xcompiler", "-fPIC",
                     "-Xcompiler", "-fvisibility=hidden", "-DBMO_BUILDING_SHARED", f"-I{ROOT}/include"]
CXX_FLAGS = ["-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-ffp-contract=off", "-Wall",
             "-DBMO_BUILDING_SHARED", f"-I{CUDA_INC}", f"-I{ROOT}/include"]


def _sources():
    cu = sorted(glob.glob(os.path.join(CSRC, "**", "*.cu"), recursive=True))
    cpp = sorted(glob.glob(os.path.join(CSRC, "**", "*.cpp"), recursive=True))
    return cu, cpp


def _headers():
    hs = glob.glob(os.path.join(CSRC, "**", "*.h"), recursive=True)
    hs += glob.glob(os.path.join(CSRC, "**", "*.cuh"), recursive=True)
    hs += glob.glob(os.path.join(ROOT, "include", "*.h"))
    return hs


def _obj_path(src: str) -> str:
    rel = os.path.relpath(src, CSRC).replace(os.sep, "__")
    return os.path.join(OBJ, rel + ".o")


def _stale(src: str, obj: str, newest_header: float) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return os.path.getmtime(src) > t or newest_header > t


def _compile(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return r.stderr


def _torch_dir():
    """Where torch is installed, found without importing it; None: it is not."""
    spec = importlib.util.find_spec("torch")
    return list(spec.submodule_search_locations)[0] if spec and spec.submodule_search_locations else None


def binding_path():
    """The torch binding for this torch, this Python and these sources: its file, built or not.
    None where it cannot be built: no torch, a torch without CUDA, or no headers."""
    t, py = _torch_dir(), sysconfig.get_paths()["include"]
    if t is None:
        return None
    needs = [os.path.join(t, "include", "c10", "cuda", "CUDAGuard.h"), os.path.join(t, "lib", "libc10_cuda.so"),
             os.path.join(t, "version.py"), os.path.join(py, "Python.h"), os.path.join(CUDA_INC, "cuda_runtime_api.h")]
    if not all(os.path.isfile(n) for n in needs):
        return None
    tag = hashlib.sha256(str(sysconfig.get_config_var("SOABI")).encode())
    for f in (needs[2], BINDING_SRC, os.path.join(ROOT, "include", "bmo_kernels.h")):
        with open(f, "rb") as src:
            tag.update(src.read())
    return os.path.join(HERE, "lib", f"_paged.{tag.hexdigest()[:12]}.so")


def build_binding(force: bool = False):
    """Builds the torch binding unless its file is there; None where it cannot be built."""
    so = binding_path()
    if so is None or (os.path.exists(so) and not force):
        return so
    t, py = _torch_dir(), sysconfig.get_paths()["include"]
    os.makedirs(os.path.dirname(so), exist_ok=True)
    tmp = f"{so}.{os.getpid()}.tmp"
    _compile([CXX, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-Wall", f"-I{ROOT}/include",
              f"-I{t}/include", f"-I{t}/include/torch/csrc/api/include", f"-I{py}", f"-I{CUDA_INC}", BINDING_SRC, "-o", tmp,
              f"-L{t}/lib", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"])
    os.replace(tmp, so)
    return so


def build(force: bool = False, jobs: int = 0, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    cu, cpp = _sources()
    live = {_obj_path(s) for s in cu + cpp}
    for o in glob.glob(os.path.join(OBJ, "*.o")):  # objects of sources that no longer exist
        if o not in live:
            os.remove(o)
    newest = max((os.path.getmtime(h) for h in _headers()), default=0.0)
    cmds = []
    objs = []
    for s in cu:
        o = _obj_path(s)
        objs.append(o)
        if force or _stale(s, o, newest):
            cmds.append([NVCC] + NVCC_FLAGS + ["-c", s, "-o", o])
    for s in cpp:
        o = _obj_path(s)
        objs.append(o)
        if force or _stale(s, o, newest):
            cmds.append([CXX] + CXX_FLAGS + ["-c", s, "-o", o])
    if cmds:
        jobs = jobs or min(len(cmds), os.cpu_count() or 4)
        with cf.ThreadPoolExecutor(jobs) as ex:
            for err in ex.map(_compile, cmds):
                if verbose and err:
                    sys.stderr.write(err)
    lib_time = os.path.getmtime(LIB) if os.path.exists(LIB) else -1.0
    if cmds or force or lib_time < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        _compile([NVCC] + ARCH + ["-shared", "-ccbin", CXX, "-o", tmp] + objs +
                 ["-cudart", "static", "-lpthread", "-ldl", "-Xlinker", "--no-undefined"])
        os.replace(tmp, LIB)
    binding = build_binding(force)
    for old in glob.glob(os.path.join(HERE, "lib", "_paged*.so")):  # of sources or versions that are no more
        if old != binding:
            os.remove(old)
    return LIB


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=0)
    ap.add_argument("-v", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.j, a.v))


if __name__ == "__main__":
    main()
