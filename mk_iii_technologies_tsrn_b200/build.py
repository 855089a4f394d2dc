"""Build recipe for the in-tree CUDA library ``_tropical_b200.so`` (sm_100a).

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` only and links them
into one shared library next to this file.  The library exposes the C ABI
declared in ``include/tropical_b200.h``; Python reaches it through ctypes
(``_lib.py``).  ``csrc/torch_host.cpp``, the host side of the language-model
operators over that ABI (outputs, workspaces, autograd nodes), becomes the Python
module ``_tropical_b200_torch.so`` beside it.  Rebuilds only what is older than
its sources and headers, and the host module for another torch or Python.  Run
``python -m mk_iii_technologies_tsrn_b200.build`` or call :func:`build`.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_NAME = "_tropical_b200.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
BUILD_DIR = os.path.join(PKG_DIR, "_build")
HOST_SOURCE = os.path.join(CSRC, "torch_host.cpp")
HOST_MODULE = "_tropical_b200_torch"
HOST_PATH = os.path.join(PKG_DIR, HOST_MODULE + ".so")
HOST_STAMP = os.path.join(BUILD_DIR, HOST_MODULE + ".for")   # what the module was compiled against

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the tropical CUDA library cannot be built")


def _sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return (
        _sources()
        + glob.glob(os.path.join(CSRC, "*.cuh"))
        + glob.glob(os.path.join(INCLUDE, "*.h"))
        + [os.path.abspath(__file__)]
    )


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    lib_mtime = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(p) > lib_mtime for p in _deps())


def _host_target() -> str:
    """The torch and Python whose headers and ABI the host module is compiled against."""
    from importlib import metadata

    try:
        version = metadata.version("torch")
    except metadata.PackageNotFoundError:      # a torch that was not installed as a package
        import torch

        version = torch.__version__
    return f"torch {version} {sys.implementation.cache_tag}\n"


def needs_host_build() -> bool:
    if not os.path.exists(HOST_PATH) or not os.path.exists(HOST_STAMP):
        return True
    with open(HOST_STAMP) as f:
        if f.read() != _host_target():
            return True
    built = os.path.getmtime(HOST_PATH)
    return any(os.path.getmtime(p) > built for p in
               [HOST_SOURCE, os.path.abspath(__file__), *glob.glob(os.path.join(INCLUDE, "*.h"))])


def build_host(verbose: bool = False) -> str:
    """Compile ``torch_host.cpp`` against the installed torch and link it to the library."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"],
                os.path.join(cuda, "include"), INCLUDE]
    tmp = HOST_PATH + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-DTORCH_EXTENSION_NAME={HOST_MODULE}", *(f"-isystem{i}" for i in includes),
           HOST_SOURCE, "-o", tmp, f"-L{libs}", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10",
           "-lc10_cuda", "-ltorch_python", f"-L{PKG_DIR}", f"-l:{LIB_NAME}",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"the host module failed to build:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, HOST_PATH)
    os.makedirs(BUILD_DIR, exist_ok=True)
    with open(HOST_STAMP, "w") as f:
        f.write(_host_target())
    return HOST_PATH


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False,
          extra_flags: list[str] | None = None, lib_path: str | None = None,
          build_dir: str | None = None) -> str:
    """Compile the library and its host module if needed and return the library's path.

    ``extra_flags`` (e.g. ``-DTP_TMA_TM=8``) and ``lib_path``/``build_dir`` build a
    variant library elsewhere without touching the in-tree one."""
    out_path = lib_path or LIB_PATH
    bdir = build_dir or BUILD_DIR
    if lib_path is None and not force and not needs_build():
        if needs_host_build():
            build_host(verbose)
        return LIB_PATH
    nvcc = _nvcc()
    os.makedirs(bdir, exist_ok=True)
    objs = []
    procs = []
    for src in _sources():
        obj = os.path.join(bdir, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, *(extra_flags or []), "-I", INCLUDE, "-c", src,
               "-o", obj]
        if ptxas_verbose:
            cmd[1:1] = ["-Xptxas", "-v"]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = []
    for src, proc in procs:
        out, _ = proc.communicate()
        text = out.decode(errors="replace")
        if proc.returncode != 0:
            failed.append((src, text))
        elif (verbose or ptxas_verbose) and text.strip():
            print(text, flush=True)
    if failed:
        msg = "\n".join(f"--- {s}\n{t}" for s, t in failed)
        raise RuntimeError(f"nvcc failed:\n{msg}")
    tmp = out_path + ".tmp"
    link = [nvcc, *ARCH_FLAGS, "-shared", "-o", tmp, *objs, "-lcudart"]
    if verbose:
        print(" ".join(link), flush=True)
    res = subprocess.run(link, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out_path)
    if lib_path is None and (force or needs_host_build()):
        build_host(verbose)
    return out_path


if __name__ == "__main__":
    force = "--force" in sys.argv
    print(build(force=force, verbose="-v" in sys.argv, ptxas_verbose="--ptxas" in sys.argv))
