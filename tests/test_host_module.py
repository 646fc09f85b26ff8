"""The extension module of actcomp.norm and actcomp.mx4 is needed by their calls
alone: without it, or with a library that lacks their entry points, the rest of
the package imports and works as before.  Runs copies of the package in child
processes."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import PKG


def package(tmp_path):
    """A copy of the package's Python files; the library comes by ACTCOMP_LIBRARY."""
    dst = tmp_path / "actcomp"
    shutil.copytree(os.path.join(PKG, "actcomp"), dst, ignore=shutil.ignore_patterns("*.so", "__pycache__"))
    return dst


def run(tmp_path, code, library=None, **env):
    full = {**os.environ, "PYTHONPATH": str(tmp_path),
            "ACTCOMP_LIBRARY": library or os.path.join(PKG, "actcomp", "libactcomp.so"), **env}
    if "ACTCOMP_AUTOBUILD" not in env:
        full.pop("ACTCOMP_AUTOBUILD", None)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=full, cwd=tmp_path, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


REST = """
import torch, actcomp
from actcomp import core, mx4, nf4, norm, offload, refcompat
assert callable(actcomp.encode) and callable(nf4.dequantize_4bit)
"""


def test_package_imports_without_the_module(tmp_path):
    package(tmp_path)
    out = run(tmp_path, REST + """
for call in (lambda: actcomp.dropout(torch.zeros(2, 8), 0.1, 0), lambda: mx4.quantize(torch.zeros(2, 32))):
    try:
        call()
        raise SystemExit("no error")
    except ImportError as e:
        print(e)
""")
    assert out.count("build it with") == 2


def test_autobuild_builds_a_missing_module(tmp_path):
    package(tmp_path)
    run(tmp_path, REST + f"""
import os, shutil
from actcomp import build
made = []
def build_host(force=False):
    here = build.host_path()
    shutil.copy(os.path.join({os.path.join(PKG, "actcomp")!r}, os.path.basename(here)), here)
    made.append(here)
    return here
build.build_host = build_host
for _ in range(2):
    try:
        actcomp.layer_norm(torch.zeros(2, 8))
        raise SystemExit("no error")
    except ValueError:  # the module's own refusal of a CPU tensor
        pass
assert len(made) == 1
""", ACTCOMP_AUTOBUILD="1")


def test_module_of_another_torch_is_not_taken(monkeypatch):
    import torch

    from actcomp import build

    here = build.build_host()
    assert os.path.exists(here)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.host_path() != here and not os.path.exists(build.host_path())


def test_library_without_the_entry_points(tmp_path):
    """An earlier build of the library (the same ABI version) serves the rest."""
    if shutil.which("gcc") is None:
        pytest.skip("gcc not found")
    from actcomp import _lib

    later = ("actcomp_dropout", "actcomp_layer_norm", "actcomp_mx4_", "actcomp_selftest_row_waits")
    names = [n for n in _lib.SIGNATURES if not n.startswith(later)]
    src = "".join(f"int {n}(void) {{ return {_lib.ABI_VERSION if n == 'actcomp_abi_version' else 0}; }}\n" for n in names)
    (tmp_path / "old.c").write_text(src)
    old = str(tmp_path / "old.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", str(tmp_path / "old.c"), "-o", old], check=True)
    package(tmp_path)
    out = run(tmp_path, REST + f"""
import os, shutil
from actcomp import build
here = build.host_path()
shutil.copy(os.path.join({os.path.join(PKG, "actcomp")!r}, os.path.basename(here)), here)
try:
    actcomp.dropout(torch.zeros(2, 8), 0.1, 0)
    raise SystemExit("no error")
except ImportError as e:
    print(e)
""", library=old)
    assert "lacks actcomp_dropout" in out
