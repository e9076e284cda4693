"""The build's steps without their compilers: what is made where torch is missing, or its module does not compile."""
import os
import subprocess
import sys

import pytest

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ops-sparse_amd", "ops_sparse",
                     "build.py")

# Runs build.py by its path, as a C caller does, with a compiler that writes its output's name into it.
SCRIPT = """
import importlib.util, os, subprocess, sys
path, folder, torch, broken = sys.argv[1:5]
if torch == "no":
    sys.modules["torch"] = None  # import raises, as where it is not installed
spec = importlib.util.spec_from_file_location("build", path)
build = importlib.util.module_from_spec(spec)
spec.loader.exec_module(build)
build.OBJ_DIR, build.OUT = os.path.join(folder, "obj"), os.path.join(folder, "library.so")
build.TORCH_OUT = os.path.join(folder, "module.so")

def run(cmd, **kw):
    if broken != "none" and any(a.endswith(broken) for a in cmd):
        return subprocess.CompletedProcess(cmd, 1, "", "broken")
    with open(cmd[cmd.index("-o") + 1], "w") as f:
        f.write(" ".join(cmd))
    return subprocess.CompletedProcess(cmd, 0, "", "")

build.subprocess.run = run
try:
    build.build_library()
except RuntimeError as e:
    sys.exit(f"RuntimeError: {e}")
"""


def build(folder, torch="yes", broken="none"):
    return subprocess.run([sys.executable, "-c", SCRIPT, BUILD, str(folder), torch, broken], capture_output=True,
                          text=True)


def test_both_are_built(tmp_path):
    res = build(tmp_path)
    assert res.returncode == 0, res.stderr
    assert "libaclsparse" not in (tmp_path / "module.so").read_text()
    assert "hipcc" in (tmp_path / "library.so").read_text()


def test_the_library_needs_no_torch(tmp_path):
    res = build(tmp_path, torch="no")
    assert res.returncode == 0, res.stderr
    assert (tmp_path / "library.so").exists() and not (tmp_path / "module.so").exists()
    assert "torch" not in (tmp_path / "library.so").read_text()


def test_a_module_that_does_not_compile_leaves_the_library_and_raises(tmp_path):
    (tmp_path / "module.so").write_text("an older one")
    res = build(tmp_path, broken="experts_torch.cpp")
    assert res.returncode != 0 and "RuntimeError" in res.stderr
    assert (tmp_path / "library.so").exists()
    assert (tmp_path / "module.so").read_text() == "an older one"


@pytest.mark.parametrize("source", ["experts_route.hip", "spmv_host.cpp"])
def test_a_source_that_does_not_compile_raises(tmp_path, source):
    res = build(tmp_path, broken=source)
    assert res.returncode != 0 and "RuntimeError" in res.stderr and not (tmp_path / "library.so").exists()
