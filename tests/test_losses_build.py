"""What the compilers see of the losses on logits, without a GPU."""

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
