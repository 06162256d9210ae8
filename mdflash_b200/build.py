"""Builds libddtree_b200.so (the C-ABI library) from csrc/*.cu for sm_100a with nvcc, and _bind.so
(the Python binding of the entry points with short kernels) from csrc/bind.cpp.

Both are built in-tree, next to this file, so they travel with the repository.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_NAME = "libddtree_b200.so"
BIND_NAME = "_bind.so"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    if os.path.exists(cand):
        return cand
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found: the ddtree_b200 CUDA library cannot be built")
    return found


def library_path() -> str:
    return os.path.join(HERE, LIB_NAME)


def binding_path() -> str:
    return os.path.join(HERE, BIND_NAME)


def binding_source() -> str:
    return os.path.join(HERE, "csrc", "bind.cpp")


def binding_commands(obj: str, out: str) -> tuple[list[str], list[str]]:
    """Compile and link commands of the binding, against the installed torch and the library."""
    import torch
    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    include = [os.path.join(home, "include"),
               os.path.join(home, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    compile_ = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-Wall",
                f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                "-I", os.path.join(HERE, "..", "include"),
                *(f for d in include for f in ("-isystem", d)), "-c", binding_source(), "-o", obj]
    libs = os.path.join(home, "lib")
    link = [compile_[0], "-shared", obj, "-o", out, "-L", HERE, "-l:" + LIB_NAME, "-L", libs,
            "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN",
            "-Wl,-rpath," + libs]
    return compile_, link


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu")))


def headers() -> list[str]:
    return (sorted(glob.glob(os.path.join(HERE, "csrc", "*.cuh"))) +
            sorted(glob.glob(os.path.join(HERE, "..", "include", "*.h"))))


def needs_build() -> bool:
    built = [library_path(), binding_path()]
    if not all(os.path.exists(f) for f in built):
        return True
    t = min(os.path.getmtime(f) for f in built)
    return any(os.path.getmtime(f) > t for f in sources() + headers() + [binding_source()])


def build(force: bool = False, verbose: bool = False) -> str:
    lib = library_path()
    if not force and not needs_build():
        return lib
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src).replace(".cu", ".o"))
        cmd = [nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    bind_obj, bind_tmp = os.path.join(objdir, "bind.o"), binding_path() + ".tmp"
    compile_, link = binding_commands(bind_obj, bind_tmp)
    procs.append((binding_source(), subprocess.Popen(compile_, stdout=subprocess.PIPE,
                                                     stderr=subprocess.STDOUT)))
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"the compiler failed on {src}:\n{out.decode()}")
        if verbose and out:
            print(out.decode())
    tmp = lib + ".tmp"
    cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", tmp, *objs]
    subprocess.run(cmd, check=True)
    os.replace(tmp, lib)
    subprocess.run(link, check=True)
    os.replace(bind_tmp, binding_path())
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
