"""CPU tests of the build: what `make` builds with and without torch, and that the torch module is not loaded into a
Python or torch that it was not built for.  Nothing is compiled here."""
import os
import re
import subprocess
import sys
import sysconfig

import pytest
import torch

import b200lab

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "turing-sm75_b200")


def _plan(*args):
    """What a full build would run."""
    r = subprocess.run(["make", "-C", PKG, "-n", "-B", *args], capture_output=True, text=True, timeout=60)
    return r.returncode, r.stdout + r.stderr


def _bare_python(tmp_path):
    """An interpreter that has no torch."""
    env = str(tmp_path / "bare")
    subprocess.run([sys.executable, "-m", "venv", "--without-pip", env], check=True, timeout=120)
    python = os.path.join(env, "bin", "python")
    assert subprocess.run([python, "-c", "import torch"], capture_output=True, timeout=60).returncode != 0
    return python


def test_a_python_without_torch_builds_the_library_and_the_tools(tmp_path):
    for python in (_bare_python(tmp_path), str(tmp_path / "none" / "python3")):
        rc, out = _plan(f"PYTHON={python}")
        assert rc == 0, out
        assert "lib/libb200lab.so" in out and "-o bin/attn_sm100" in out and "-o bin/gdn_sm100" in out
        assert "torch_kv8.cpp" not in out
        rc, out = _plan("lib/_b200torch.so", f"PYTHON={python}")  # asked for by name: it says why not
        assert "has no torch" in out


def test_a_python_with_torch_builds_the_module_for_itself():
    rc, out = _plan(f"PYTHON={sys.executable}")
    assert rc == 0 and "csrc/torch_kv8.cpp" in out and "-o bin/attn_sm100" in out, out
    line = [x for x in out.replace("\\\n", " ").splitlines() if "-o lib/_b200torch.so" in x][0]
    for d in re.findall(r"-(?:I|isystem |L)\s*(/\S+)", line):
        assert os.path.isdir(d), d
    root = os.path.dirname(torch.__file__)
    assert f"-isystem {root}/include" in line and f"-L{root}/lib" in line


@pytest.mark.parametrize("built", ["cpython-39-x86_64-linux-gnu " + str(torch.__version__),
                                   sysconfig.get_config_var("SOABI") + " 1.0.0", ""])
def test_a_module_of_another_python_or_torch_is_not_loaded(tmp_path, monkeypatch, built):
    (tmp_path / "lib").mkdir()
    (tmp_path / "lib" / "_b200torch.so").write_bytes(b"not to be loaded")
    (tmp_path / "lib" / "_b200torch.txt").write_text(built + "\n")
    b200lab.lib()
    monkeypatch.setattr(b200lab, "_HERE", str(tmp_path))
    monkeypatch.setattr(b200lab, "_NATIVE", None)
    with pytest.raises(ImportError, match="was built for"):
        b200lab._native()


def test_the_module_as_built_is_loaded():
    assert b200lab._native().append
