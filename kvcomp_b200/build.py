"""Compile kvcomp_b200/csrc/*.cu into kvcomp_b200/lib/libkvcomp_b200.so for sm_100a, and kvcomp_b200/csrc/kvc_torch.cpp, the paged cache's calls for torch, into
kvcomp_b200/lib/kvc_torch.<torch's version, Python's tag, ABI>.so.

    python -m kvcomp_b200.build [--force] [--verbose] [--library]          # --library: the library alone, which needs no torch

nvcc cross-compiles without a GPU.  The library is kept in-tree so that it ships with the
source snapshot; it is rebuilt when any source is newer than it.
"""
import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libkvcomp_b200.so")
BINDING_SOURCE = os.path.join(CSRC, "kvc_torch.cpp")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "--expt-extended-lambda", "-shared", "-Xcompiler", "-fPIC", "-cudart", "shared"]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def is_stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(f) > t for f in _deps())


def binding_path():
    """Where the binding for this torch and this Python lies: it is compiled against the classes of the one and the headers of the other."""
    import torch
    return os.path.join(LIB_DIR, "kvc_torch.%s.%s.abi%d.so" % (torch.__version__, sysconfig.get_config_var("SOABI"), torch._C._GLIBCXX_USE_CXX11_ABI))


def binding_is_stale():
    path = binding_path()
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(f) > t for f in [BINDING_SOURCE] + glob.glob(os.path.join(INCLUDE, "*.h")))


def _run(cmd, to, verbose):
    """Run a compiler that writes `to`.  It writes beside it first: a process that starts meanwhile sees the old file or the new one."""
    made = "%s.%d.tmp" % (to, os.getpid())
    r = subprocess.run(cmd + ["-o", made], capture_output=True, text=True)
    if verbose:
        sys.stderr.write(r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError("%s failed:\n%s\n%s" % (os.path.basename(cmd[0]), " ".join(cmd), r.stderr[-4000:]))
    os.replace(made, to)
    return to


def build_binding(force=False, verbose=False):
    import torch
    path = binding_path()
    if not force and not binding_is_stale():
        return path
    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    os.makedirs(LIB_DIR, exist_ok=True)
    compiler = shutil.which(os.environ.get("CXX", "g++"))
    if not compiler:
        raise RuntimeError("no C++ compiler found; kvc_torch cannot be built")
    cmd = [compiler, "-std=c++17", "-O2", "-shared", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI]
    for d in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"]):
        cmd += ["-isystem", d]
    cmd += [BINDING_SOURCE, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    return _run(cmd, path, verbose)


def nvcc_path():
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found; libkvcomp_b200.so cannot be built")


def build(force=False, verbose=False, binding=True):
    """The library, and then the binding where there is torch to bind to.  Each is left as it is where nothing is newer."""
    if force or is_stale():
        os.makedirs(LIB_DIR, exist_ok=True)
        _run([nvcc_path()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + sources(), LIB, verbose)
    if binding:
        if importlib.util.find_spec("torch") is not None:
            build_binding(force, verbose)
        else:
            sys.stderr.write("no torch here: kvc_torch, through which kvcomp_b200.ops makes the paged cache's calls, is not built\n")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, binding="--library" not in sys.argv))
