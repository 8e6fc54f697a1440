"""
Build ``libnunchaku_b200.so`` from ``csrc/*.cu`` with nvcc for sm_100a, in-tree.

``python -m nunchaku_rocm_b200.build`` (or :func:`build`) compiles every translation unit whose
object is older than its sources and links one shared library next to this file.  nvcc
cross-compiles without a GPU, so this also runs on a CPU-only machine.

``csrc/binding/*.cpp`` (torch's side of the differentiable operators: plain C++ against torch's headers) becomes the
extension module ``_binding`` beside it, rebuilt too when torch or Python has another version.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libnunchaku_b200.so")
BINDING = os.path.join(HERE, "_binding.so")

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or add it to PATH")


def _newest(paths) -> float:
    return max(os.path.getmtime(p) for p in paths)


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _binding_stamp() -> str:
    return os.path.join(OBJ, "binding.versions")


def _binding_versions() -> str:
    import torch

    return f"torch {torch.__version__} python {sys.version.split()[0]}"


def _binding_command(force: bool) -> list[str] | None:
    """The compiler's command for the torch binding, or ``None`` where it is up to date."""
    import sysconfig

    import torch

    src = sorted(os.path.join(CSRC, "binding", f) for f in os.listdir(os.path.join(CSRC, "binding")) if f.endswith(".cpp"))
    newest = _newest([*src, os.path.join(os.path.dirname(HERE), "include", "nunchaku_b200.h")])
    stamp = _binding_stamp()
    made = open(stamp).read() if os.path.exists(stamp) else ""
    if not force and os.path.exists(BINDING) and os.path.getmtime(BINDING) >= newest and made == _binding_versions():
        return None
    # the compiler that nvcc takes too, whatever $CXX is: one that links a C++ library of its own in brings a second copy of
    # its locale into torch's process, and the first number printed into an error message ends it
    cxx = shutil.which("g++")
    if cxx is None:
        raise RuntimeError("g++ not found on PATH")
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    return [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in include), *src,
            f"-L{os.path.join(root, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-o", BINDING]


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile and link; returns the library path."""
    nvcc = _nvcc()
    os.makedirs(OBJ, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(os.path.join(os.path.dirname(HERE), "include", "nunchaku_b200.h"))
    dep_time = _newest(headers)
    jobs = []
    objs = []
    for src in sources():
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), dep_time):
            jobs.append([nvcc, *NVCC_FLAGS, "-c", src, "-o", obj])

    binding = _binding_command(force)
    if binding:
        jobs.append(binding)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr)

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        list(ex.map(run, jobs))
    if binding:
        with open(_binding_stamp(), "w") as f:
            f.write(_binding_versions())
    if [j for j in jobs if j is not binding] or not os.path.exists(LIB) or os.path.getmtime(LIB) < _newest(objs):
        run([nvcc, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
