"""The losses on logits in the index-checked build (libmoteopt_checked.so): no index check fails, and the outputs equal the
release library's bit for bit."""

import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def _run(lib: Path, out: Path) -> int:
    env = dict(os.environ, MOTEOPT_LIB=str(lib))
    r = subprocess.run([sys.executable, str(ROOT / "tests" / "losses_workload.py"), str(out)], env=env, capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    return int(r.stdout.strip().splitlines()[-1].split()[1])


def test_checked_build_finds_no_bad_index_and_matches_the_release_build(tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    checked = ROOT / "mote_b200" / "libmoteopt_checked.so"
    assert checked.exists(), "build it with `python -m mote_b200.build --checked` (__graft_entry__.build does)"
    assert _run(checked, tmp_path / "checked.npz") == 0
    assert _run(ROOT / "mote_b200" / "libmoteopt.so", tmp_path / "release.npz") == 0
    x, y = np.load(tmp_path / "checked.npz"), np.load(tmp_path / "release.npz")
    assert sorted(x.files) == sorted(y.files)
    for k in x.files:   # bit for bit (NaN-safe)
        assert np.array_equal(x[k].view(np.uint32), y[k].view(np.uint32)), k
