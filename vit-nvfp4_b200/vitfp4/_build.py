"""Build libvitfp4.so (the sm_100a CUDA kernels + C ABI) in-tree with nvcc.

    python -m vitfp4._build            # or vitfp4._build.build()

The library lands next to this file (``vitfp4/libvitfp4.so``) so it travels with the
source tree; it is rebuilt only when a source or header is newer than the library.  Beside it
``vitfp4/_fast.so``, a host-side module (g++, torch's headers) that makes the plain calls of the small
ops without the Python argument path; without it those calls take that path to the same kernels.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import warnings

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(PKG), "csrc")
INCLUDE = os.path.join(os.path.dirname(os.path.dirname(PKG)), "include")
LIB = os.path.join(PKG, "libvitfp4.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or install the CUDA toolkit")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(INCLUDE, "*.h"))


FAST_SRC = os.path.join(CSRC, "host", "vf4_fast.cpp")
FAST = os.path.join(PKG, "_fast.so")


def fast_built_for() -> str:
    """What the module is compiled against, as it names it itself (``built_for``): torch's C++ interface holds for one
    release.  The module is neither kept nor loaded beside another."""
    import torch
    return f"vf4_fast for torch {torch.__version__}, python {sys.version_info[0]}.{sys.version_info[1]}"


def _fast_is_current() -> bool:
    deps = [FAST_SRC, os.path.join(INCLUDE, "vitfp4.h")]
    if not os.path.exists(FAST) or any(os.path.getmtime(d) > os.path.getmtime(FAST) for d in deps):
        return False
    with open(FAST, "rb") as f:
        return fast_built_for().encode() + b"\0" in f.read()


def _fast_command(out: str) -> list[str]:
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DVF4_BUILT_FOR="{fast_built_for()}"',
            *[f for p in inc for f in ("-isystem", p)], "-I", INCLUDE, FAST_SRC, "-o", out,
            "-L", PKG, "-l:libvitfp4.so", "-Wl,-rpath,$ORIGIN", "-L", os.path.join(root, "lib"),
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def build_fast(force: bool = False) -> str | None:
    """Compile csrc/host/vf4_fast.cpp against torch and libvitfp4.so; returns the module's path.  Where that cannot be
    done (no g++, no headers) it warns and returns None, with no older module left behind: the calls work without."""
    if not force and _fast_is_current():
        return FAST
    tmp = FAST + ".tmp"
    try:
        r = subprocess.run(_fast_command(tmp), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        why = r.stdout if r.returncode else None
    except (OSError, RuntimeError) as e:   # no g++, no CUDA toolkit
        why = str(e)
    if why is not None:
        if os.path.exists(FAST):
            os.remove(FAST)
        warnings.warn(f"vitfp4/_fast.so was not built; plain calls of the small ops take the Python path: {why}",
                      stacklevel=2)
        return None
    os.replace(tmp, FAST)
    return FAST


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(d) <= t for d in _deps())


def build(force: bool = False, verbose: bool = False, jobs: int | None = None) -> str:
    """Compile every csrc/*.cu for sm_100a and link libvitfp4.so; returns its path."""
    if not force and up_to_date():
        build_fast()
        return LIB
    nvcc = _nvcc()
    objdir = os.path.join(os.path.dirname(PKG), "_build")
    os.makedirs(objdir, exist_ok=True)
    objs, procs = [], []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    failed = []
    for src, pr in procs:
        out, _ = pr.communicate()
        if verbose or pr.returncode:
            sys.stderr.write(out)
        if pr.returncode:
            failed.append(src)
    if failed:
        raise RuntimeError(f"nvcc failed for {failed}")
    tmp = LIB + ".tmp"
    link = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", *objs, "-o", tmp, "-lcuda"]
    r = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode:
        sys.stderr.write(r.stdout)
        raise RuntimeError("link of libvitfp4.so failed")
    os.replace(tmp, LIB)
    build_fast(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
