"""A call's result must not depend on the calls before it: sizes whose static
and dynamic shared memory together pass 48 KB while the dynamic part alone does
not, each as the first call of its kernel in a fresh process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("group", ["linear", "norm"])
def test_first_call_of_each_kernel(group):
    r = subprocess.run([sys.executable, os.path.join(HERE, "first_call_worker.py"), group], capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
