"""Build libmoteopt.so (the CUDA kernels and the C ABI of include/moteopt.h) for sm_100a and _torch_losses.so (the losses'
torch binding, host code), in-tree.

    python -m mote_b200.build            # or: python mote_b200/build.py
    python -m mote_b200.build --checked  # libmoteopt_checked.so

The release build keeps ptxas's per-kernel resource report (registers, spills, shared memory) in
mote_b200/_build/ptxas_release.txt.

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically and takes the driver's
cuTensorMapEncodeTiled through cudaGetDriverEntryPoint, so it needs no -lcuda at link time.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libmoteopt.so"
CHECKED_LIB = PKG / "libmoteopt_checked.so"   # the same library with MOTE_OPT_CHECKS: index checks in every kernel
RESOURCES = PKG / "_build" / "ptxas_release.txt"   # ptxas's per-kernel registers / spills of the release build
SOURCES = [CSRC / "moteopt.cu"]
BINDING = PKG / "_torch_losses.so"
BINDING_SOURCE = CSRC / "torch_losses.cpp"
HEADERS = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [ROOT / "include" / "moteopt.h"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = [os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"]
    for c in cand:
        if c and Path(c).exists():
            return c
    raise RuntimeError("nvcc not found (set NVCC=...)")


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in SOURCES + HEADERS)


def built_for() -> str:
    """What a binding depends on beside its sources: it uses torch's and Python's C++ objects as their headers lay them out."""
    import torch
    return f"torch {torch.__version__}, C++ ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, {sys.implementation.cache_tag}"


def binding_fits() -> bool:
    """Whether the binding is there and was built for this torch and this Python (it holds their names as its doc string)."""
    return BINDING.exists() and f"built for {built_for()}.".encode() in BINDING.read_bytes()


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """g++ the torch binding of the losses (no CUDA code; it is given libmoteopt.so's functions when it is imported)."""
    import torch
    sources = [BINDING_SOURCE, ROOT / "include" / "moteopt.h", Path(__file__).resolve()]
    if not force and binding_fits() and all(p.stat().st_mtime <= BINDING.stat().st_mtime for p in sources):
        return BINDING
    from torch.utils import cpp_extension as ext
    tmp = BINDING.with_suffix(".so.tmp")
    inc = [str(ROOT / "include"), sysconfig.get_paths()["include"], *ext.include_paths("cuda")]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DMOTEOPT_BUILT_FOR="{built_for()}"', *[a for d in inc for a in ("-I", d)],
           str(BINDING_SOURCE), "-o", str(tmp), *[a for d in ext.library_paths("cuda") for a in ("-L", d)], "-lc10",
           "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise subprocess.CalledProcessError(r.returncode, cmd)
    os.replace(tmp, BINDING)
    return BINDING


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None, checked: bool = False) -> Path:
    """nvcc the library, then the torch binding, which the library does not need: without torch or a host compiler it is left
    out with a message. `checked` builds libmoteopt_checked.so, which counts failed index checks (moteopt_check_count), instead
    of the two."""
    if checked:
        return build_library(CHECKED_LIB, verbose, extra)
    if force or needs_build():
        build_library(LIB, verbose, extra)
    try:
        build_binding(force, verbose)
    except Exception as e:
        BINDING.unlink(missing_ok=True)   # not the one of another library
        sys.stderr.write(f"{LIB.name} is built; {BINDING.name} is not, so mote_b200's losses cannot be called: {e}\n")
    return LIB


def build_library(out: Path, verbose: bool = False, extra: list[str] | None = None) -> Path:
    """nvcc LIB or CHECKED_LIB."""
    checked = out == CHECKED_LIB
    if checked:
        extra = ["-DMOTE_OPT_CHECKS", *(extra or [])]
    else:   # keep ptxas's resource report (registers, spills, shared memory per kernel) beside the build
        extra = ["-Xptxas", "-v", *(extra or [])]
    tmp = out.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC,-fvisibility=hidden",
           "-I", str(ROOT / "include"), "-I", str(CSRC), "--expt-relaxed-constexpr", "-o", str(tmp),
           *[str(s) for s in SOURCES], *(extra or [])]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise subprocess.CalledProcessError(r.returncode, cmd)
    if not checked:
        RESOURCES.parent.mkdir(exist_ok=True)
        RESOURCES.write_text(r.stderr + r.stdout)
    elif verbose:
        sys.stderr.write(r.stderr)
    os.replace(tmp, out)
    return out


if __name__ == "__main__":
    v = "-v" in sys.argv
    print(build(force=True, verbose=v, checked="--checked" in sys.argv))
