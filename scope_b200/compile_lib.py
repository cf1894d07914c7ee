"""Compile libscope_b200.so (the C-ABI library) in-tree with nvcc for sm_100a, and _binding.so (the CPython binding of
the paged cache's entries) with the host compiler.

    python -m scope_b200.compile_lib [-v]

Objects are compiled in parallel into scope_b200/_build/ and linked with the
static CUDA runtime; the library links nothing from PyTorch.  The binding is
compiled against PyTorch's headers and resolves its symbols from the PyTorch
that the process has loaded.
"""
from __future__ import annotations

import concurrent.futures as cf
import contextlib
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libscope_b200.so")
BINDING_SRC = os.path.join(CSRC, "binding.cpp")
BINDING = os.path.join(PKG, "_binding.so")
BINDING_STAMP = os.path.join(BUILD, "binding.stamp")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr",
              "-Xptxas", "-v", "-I" + INCLUDE, "-I" + CSRC]


def nvcc() -> str:
    for cand in (os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc"), shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers_mtime() -> float:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, verbose: bool) -> tuple[str, str]:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", src, "-o", obj]
    # nvcc picks the host compiler from PATH; the system gcc links OpenMP-free C++ fine.
    env = dict(os.environ)
    env.pop("CC", None)
    env.pop("CXX", None)
    out = subprocess.run(cmd, capture_output=True, text=True, env=env)
    if out.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{out.stdout}\n{out.stderr}")
    return obj, out.stderr if verbose else ""


def binding_stamp() -> str:
    """What the binding is compiled against beside its sources: it holds PyTorch's and Python's C++ layouts."""
    import torch
    return "\n".join([torch.__version__, str(torch.version.git_version), os.path.dirname(torch.__file__),
                      f"cxx11 abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}", sys.version, sysconfig.get_paths()["include"]])


def build_binding(verbose: bool = False, force: bool = False) -> str:
    """Build the binding if its source is newer than it, or if it was built against another PyTorch or Python; return its
    path."""
    newest = max(os.path.getmtime(BINDING_SRC), _headers_mtime())
    stamp = binding_stamp()
    if not force and os.path.exists(BINDING) and os.path.getmtime(BINDING) >= newest and os.path.exists(BINDING_STAMP):
        with open(BINDING_STAMP) as f:
            if f.read() == stamp:
                return BINDING
    import torch
    root = os.path.dirname(torch.__file__)
    cxx = shutil.which("g++")
    if cxx is None:
        raise RuntimeError("g++ not found")
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", "-Wno-sign-compare",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I" + INCLUDE, "-I" + sysconfig.get_paths()["include"], "-isystem", os.path.join(root, "include"),
           "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-isystem", os.path.join(cuda, "include"), BINDING_SRC, "-o", BINDING + ".tmp",
           "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-lc10_cuda", "-lc10"]
    out = subprocess.run(cmd, capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError(f"g++ failed on {BINDING_SRC}:\n{out.stdout}\n{out.stderr}")
    if verbose:
        sys.stdout.write(out.stderr)
    os.makedirs(BUILD, exist_ok=True)
    with contextlib.suppress(FileNotFoundError):
        os.remove(BINDING_STAMP)
    os.replace(BINDING + ".tmp", BINDING)
    with open(BINDING_STAMP, "w") as f:
        f.write(stamp)
    return BINDING


def build(verbose: bool = False, force: bool = False) -> str:
    """Build the library and the binding where a source is newer; return the library's path."""
    with cf.ThreadPoolExecutor(max_workers=1) as ex:
        binding = ex.submit(build_binding, verbose, force)
        lib = build_lib(verbose, force)
        binding.result()
    return lib


def build_lib(verbose: bool = False, force: bool = False) -> str:
    """Build the library if any source is newer than it; return its path."""
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    newest = max([os.path.getmtime(s) for s in srcs] + [_headers_mtime()])
    if not force and os.path.exists(LIB) and os.path.getmtime(LIB) >= newest:
        return LIB
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        results = list(ex.map(lambda s: _compile(s, verbose), srcs))
    objs = [r[0] for r in results]
    if verbose:
        for _, log in results:
            sys.stdout.write(log)
    cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", LIB + ".tmp", *objs, "-lcuda" if False else "-ldl"]
    env = dict(os.environ)
    env.pop("CC", None)
    env.pop("CXX", None)
    out = subprocess.run(cmd, capture_output=True, text=True, env=env)
    if out.returncode != 0:
        raise RuntimeError(f"link failed:\n{out.stdout}\n{out.stderr}")
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
