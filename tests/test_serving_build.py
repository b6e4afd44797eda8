"""Building and loading the serving operators' Python binding (CPU only), in
a copy of the package: what is missing or out of date is built or said, never
passed over."""

import glob
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINDING = "from grokking_abmod_b200 import ops; print(ops._binding().__name__)"


@pytest.fixture
def copy(tmp_path):
    """The package with its built files, in date."""
    from grokking_abmod_b200 import build
    build.build()
    for part in ("grokking_abmod_b200", "include"):
        shutil.copytree(os.path.join(ROOT, part), tmp_path / part, ignore=shutil.ignore_patterns("*.so", "__pycache__"))
    for built in glob.glob(os.path.join(ROOT, "grokking_abmod_b200", "*.so")):
        shutil.copy(built, tmp_path / "grokking_abmod_b200")  # newer than the sources
    return tmp_path


def _run(copy, code, **env):
    return subprocess.run([sys.executable, "-c", code], cwd=copy, env={**os.environ, **env}, capture_output=True,
                          text=True, timeout=300)


def test_the_copy_loads_as_it_is(copy):
    r = _run(copy, BINDING, CXX="/bin/false")
    assert r.returncode == 0 and "_serving" in r.stdout, r.stderr


def test_the_library_builds_without_torch(copy):
    """Callers of the C interface need the CUDA compiler only."""
    for built in glob.glob(str(copy / "grokking_abmod_b200" / "_serving*")):
        os.remove(built)
    r = _run(copy, "import sys; sys.modules['torch'] = None\n"
                   "from grokking_abmod_b200.build import build; print(build())")
    assert r.returncode == 0 and r.stdout.strip().endswith("libmeshb200.so"), r.stderr
    assert "torch" in r.stderr
    r = _run(copy, "import sys; sys.modules['torch'] = None\n"
                   "from grokking_abmod_b200 import _lib; _lib.load().mb_version")
    assert r.returncode == 0, r.stderr


def test_a_binding_that_does_not_build_is_an_error(copy):
    """Not the use of the one that was there, of older sources."""
    with open(copy / "grokking_abmod_b200" / "csrc" / "binding.cpp", "a") as f:
        f.write("// newer\n")
    r = _run(copy, BINDING, CXX="/bin/false")
    assert r.returncode != 0 and "false failed" in r.stderr, r.stdout + r.stderr
    # the library needs no binding
    r = _run(copy, "from grokking_abmod_b200 import _lib; _lib.load().mb_version", CXX="/bin/false")
    assert r.returncode == 0, r.stderr


def test_a_binding_of_another_torch_is_not_used(copy):
    r = _run(copy, "import torch; torch.__version__ = '2.0.0'\n" + BINDING, CXX="/bin/false")
    assert r.returncode != 0 and "false failed" in r.stderr, r.stdout + r.stderr


@pytest.mark.slow
def test_a_binding_does_not_meet_a_library_of_another_header(copy):
    """A library that stayed older while the binding was built: refused when
    it is loaded, before any argument structure is passed."""
    with open(copy / "include" / "meshb200.h", "a") as f:
        f.write("/* newer */\n")
    library = copy / "grokking_abmod_b200" / "libmeshb200.so"
    later = os.path.getmtime(copy / "include" / "meshb200.h") + 10
    os.utime(library, (later, later))
    r = _run(copy, BINDING)
    assert r.returncode != 0 and "ImportError" in r.stderr and "header" in r.stderr, r.stdout + r.stderr
