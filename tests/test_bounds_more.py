"""The bounds-checked build on the root-mean-square norm, the 8-bit operators and the
cross entropy: their stores check their places and record a bit instead of trapping.
Ragged shapes must leave the device error word clear, and every output must equal the
product library's bit for bit."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def run(lib, out):
    env = {k: v for k, v in os.environ.items() if k != "ACTCOMP_LIBRARY"}
    if lib:
        env["ACTCOMP_LIBRARY"] = lib
    subprocess.run([sys.executable, os.path.join(HERE, "bounds_more_worker.py"), out], check=True, env=env, timeout=600)
    return dict(np.load(out))


def test_operators_stay_in_bounds(tmp_path):
    from actcomp import _lib, build

    assert os.path.exists(build.LIB_BC), "libactcomp_bc.so is built by __graft_entry__.build()"
    checked, plain = run(build.LIB_BC, str(tmp_path / "bc.npz")), run(None, str(tmp_path / "plain.npz"))
    for r in (checked, plain):
        assert r["word"][0] == 0 and r["status"][0] == _lib.ACT_OK
    assert set(checked) == set(plain)
    for k in plain:
        assert np.array_equal(checked[k], plain[k]), k
