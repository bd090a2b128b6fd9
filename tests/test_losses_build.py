"""What the compilers see of the losses on logits, without a GPU."""

import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_what_goes_to_another_blocks_memory_is_aligned(tmp_path):
    """A part of a row is stored with one instruction of 8 bytes."""
    from mote_b200 import build
    try:
        nvcc = build.nvcc()
    except RuntimeError:
        pytest.skip("needs nvcc")
    src = tmp_path / "part.cu"
    src.write_text('#include "loss_kernels.cuh"\n'
                   "static_assert(sizeof(moteopt::loss::Part) == 8 && alignof(moteopt::loss::Part) == 8);\n")
    r = subprocess.run([nvcc, *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I", str(ROOT / "include"), "-I",
                        str(build.CSRC), "-cuda", "-o", str(tmp_path / "part.ii"), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("missing", ["a host compiler", "torch", "a header"])
def test_the_library_is_built_without_what_the_binding_needs(tmp_path, monkeypatch, capsys, missing):
    """nvcc alone builds the C library (nvcc is not run here); an older binding does not stay beside it."""
    import sys

    from mote_b200 import build
    built = []
    monkeypatch.setattr(build, "LIB", tmp_path / "libmoteopt.so")
    monkeypatch.setattr(build, "BINDING", tmp_path / "_torch_losses.so")
    monkeypatch.setattr(build, "build_library", lambda out, *a, **k: built.append(out) or out, raising=False)
    build.BINDING.write_bytes(b"of another library")
    if missing == "a host compiler":
        monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    elif missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        bad = tmp_path / "bad.cpp"
        bad.write_text('#include "no_such_header.h"\n')
        monkeypatch.setattr(build, "BINDING_SOURCE", bad)
    assert build.build(force=True) == build.LIB and built == [build.LIB]
    assert not build.BINDING.exists() and "_torch_losses.so is not" in capsys.readouterr().err


def test_a_binding_of_another_torch_is_built_again_and_not_loaded(tmp_path, monkeypatch):
    import torch

    from mote_b200 import build, losses
    binding = tmp_path / "_torch_losses.so"
    shutil.copy2(build.BINDING, binding)
    monkeypatch.setattr(build, "BINDING", binding)
    monkeypatch.setattr(losses, "BINDING", binding, raising=False)
    os.utime(binding)   # newer than every source
    kept = binding.stat().st_ino
    assert build.build_binding() == binding and binding.stat().st_ino == kept
    monkeypatch.setattr(torch, "__version__", "2.0.0+other")
    with pytest.raises(ImportError, match="built for torch 2.0.0.other"):
        losses._load()
    assert build.build_binding() == binding and binding.stat().st_ino != kept
    binding.unlink()
    with pytest.raises(ImportError, match="not found"):
        losses._load()
