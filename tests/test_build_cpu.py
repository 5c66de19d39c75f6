"""The in-tree build without a GPU: what `make` builds with and without a Python
that has torch, and for which one."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import PKG

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make")


def plan(*args):
    """What make would run, everything taken as out of date."""
    r = subprocess.run(["make", "-n", "-B", "-C", PKG, *args], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


@pytest.mark.parametrize("python", ["false", "/no/such/python"])
def test_without_python_or_torch_the_library_is_still_built(python):
    out = plan(f"PYTHON={python}")
    assert "libnelisp_cuda.so" in out and "nelisp-cuserver" in out
    assert "_serving.so" not in out


def test_an_interpreter_without_torch(tmp_path):
    """-S -I: no site-packages, as on a machine without torch."""
    exe = tmp_path / "python"
    exe.write_text(f'#!/bin/sh\nexec "{sys.executable}" -S -I "$@"\n')
    exe.chmod(0o755)
    assert "_serving.so" not in plan(f"PYTHON={exe}")


def test_a_torch_without_cuda_or_without_metadata(tmp_path):
    """Without CUDA its headers would not do; without metadata it is torch all the
    same."""
    (tmp_path / "torch" / "lib").mkdir(parents=True)
    (tmp_path / "torch" / "__init__.py").write_text("")
    exe = tmp_path / "python"
    exe.write_text(f'#!/bin/sh\nexec env PYTHONPATH="{tmp_path}" "{sys.executable}" -S "$@"\n')
    exe.chmod(0o755)
    assert "_serving.so" not in plan(f"PYTHON={exe}")
    (tmp_path / "torch" / "lib" / "libc10_cuda.so").write_text("")
    assert "_serving.so" in plan(f"PYTHON={exe}")


def test_with_torch_the_module_is_built_by_that_interpreter():
    out = plan(f"PYTHON={sys.executable}")
    line = next(x for x in out.split("\n") if "-o nelisp_cuda/_serving.so" in x)
    assert f"{sys.executable} csrc/torch_flags.py" in line


def test_another_torch_builds_the_module_anew(tmp_path):
    """The interpreter and torch it was built for are a prerequisite of it."""
    for name in ("Makefile", "csrc"):
        os.symlink(os.path.join(PKG, name), tmp_path / name)
    (tmp_path / "nelisp_cuda").mkdir()
    (tmp_path / "_build").mkdir()
    which = subprocess.run([sys.executable, os.path.join(PKG, "csrc", "torch_flags.py"), "--which"],
                           capture_output=True, text=True, check=True).stdout
    assert which.count(" ") == 2 and "torch" in which
    stamp, module = tmp_path / "_build" / "torch", tmp_path / "nelisp_cuda" / "_serving.so"

    def stale():
        os.utime(module, (2 ** 31, 2 ** 31))           # newer than its sources
        if stamp.stat().st_mtime > 2 ** 30 and stamp.read_text() == which:
            os.utime(stamp, (2 ** 30, 2 ** 30))
        r = subprocess.run(["make", "-C", str(tmp_path), "-f", "Makefile", f"PYTHON={sys.executable}",
                            "CXX=true", "NVCC=true", "_build/torch"], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return stamp.read_text()

    module.touch()
    stamp.write_text("cpython-00 /no/torch/__init__.py 0.0\n")
    assert stale() == which                            # rewritten: the module is out of date
    before = stamp.stat().st_mtime
    assert stale() == which
    assert stamp.stat().st_mtime <= before             # not written again for the same torch


def test_build_passes_its_own_interpreter(monkeypatch):
    from nelisp_cuda import build
    ran = []
    monkeypatch.setattr(build.subprocess, "run", lambda args, check: ran.append(args))
    build.build(jobs=3)
    assert f"PYTHON={sys.executable}" in ran[0] and "-j3" in ran[0]
