"""In-tree build of libactcomp.so (sm_100a) with nvcc.

``python triton-kernel-test_b200/actcomp/build.py`` (this file run on its own:
importing the ``actcomp`` package loads the library it builds) compiles every
``csrc/*.cu`` into ``actcomp/libactcomp.so`` next to this file.  The library
links the CUDA runtime statically and takes the driver's tensor-map encoder
through ``cudaGetDriverEntryPoint``, so it loads on a machine without a GPU
(the CPU test suite checks its exported symbols) and needs no libcuda at link
time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(ROOT, "csrc")
LIB = os.path.join(PKG, "libactcomp.so")
# the bounds-checked build (-DACT_BOUNDS_CHECK): device-side index checks that
# record a bit in the device error word instead of trapping; tests only
LIB_BC = os.path.join(PKG, "libactcomp_bc.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17", "-rdc=true",
    "--fmad=false",               # keep every a*b+c a separately rounded mul and add (oracle parity)
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libactcomp")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps() -> list[str]:
    hdr = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    inc = os.path.join(os.path.dirname(ROOT), "include", "actcomp.h")
    return sources() + hdr + ([inc] if os.path.exists(inc) else [])


def stale(lib: str = LIB) -> bool:
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    return any(os.path.getmtime(p) > t for p in _deps())


def host_path() -> str:
    """The extension module of the host side of actcomp.norm and actcomp.mx4
    (csrc/host.cpp).  It is compiled against one torch and one Python and named
    after both, so that one built for others is never loaded or taken as up to date."""
    import sysconfig

    import torch

    return os.path.join(PKG, f"_host-torch{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}")


def build_host(force: bool = False) -> str:
    """Compile (if stale) csrc/host.cpp against torch's headers and return the
    module's path."""
    import sysconfig

    src, out = os.path.join(CSRC, "host.cpp"), host_path()
    deps = [src, os.path.join(os.path.dirname(ROOT), "include", "actcomp.h")]
    if not force and os.path.exists(out) and all(os.path.getmtime(p) <= os.path.getmtime(out) for p in deps):
        return out
    import torch

    base = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    inc = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], cuda]
    tmp = out + ".tmp"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", src, "-o", tmp,
                    *[f"-I{i}" for i in inc], f"-L{os.path.join(base, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
                    "-ltorch", "-ltorch_python", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"],
                   check=True)
    os.replace(tmp, out)
    return out


def build(force: bool = False, verbose: bool = False, jobs: int | None = None, bounds_check: bool = False) -> str:
    """Compile (if stale) and return the path of libactcomp.so (libactcomp_bc.so
    with bounds_check)."""
    lib = LIB_BC if bounds_check else LIB
    build_host(force and not bounds_check)
    if not force and not stale(lib):
        return lib
    exe = nvcc()
    flags = NVCC_FLAGS + (["-DACT_BOUNDS_CHECK"] if bounds_check else [])
    tmp = tempfile.mkdtemp(prefix="actcomp_build_")
    try:
        objs = []
        procs = []
        for src in sources():
            obj = os.path.join(tmp, os.path.basename(src) + ".o")
            cmd = [exe, *flags, "-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
            objs.append(obj)
        failed = []
        for src, p in procs:
            out, _ = p.communicate()
            if out.strip() and (verbose or p.returncode):
                print(out, file=sys.stderr)
            if p.returncode:
                failed.append(src)
        if failed:
            raise RuntimeError(f"nvcc failed for {failed}")
        out_tmp = lib + ".tmp"
        cmd = [exe, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC", "-o", out_tmp,
               *objs, "-cudart", "static"]
        subprocess.run(cmd, check=True)
        os.replace(out_tmp, lib)
    finally:
        shutil.rmtree(tmp, ignore_errors=True)
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, bounds_check="--bounds-check" in sys.argv))
