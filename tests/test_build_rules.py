"""When objects are compiled again (no compiler runs here)."""
import os
import subprocess

import pytest

from kfold_b200 import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of two files; what the compiler was called for."""
    csrc, include = tmp_path / "pkg" / "csrc", tmp_path / "include"
    csrc.mkdir(parents=True)
    include.mkdir()
    files = {"a": csrc / "a.cu", "b": csrc / "residual_norm.cu", "header": csrc / "h.cuh", "abi": include / "kfold_b200.h", "build": tmp_path / "pkg" / "build.py"}
    for f in files.values():
        f.write_text("")
        os.utime(f, (1000, 1000))
    calls = []

    def run(cmd, **more):
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w"):
            pass
        os.utime(out, (2000, 2000))
        calls.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B, "PKG", str(tmp_path / "pkg"))
    monkeypatch.setattr(B, "CSRC", str(csrc))
    monkeypatch.setattr(B, "OUT_DIR", str(tmp_path / "pkg" / "_C"))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "pkg" / "_C" / "lib.so"))
    monkeypatch.setattr(B, "__file__", str(files["build"]))
    monkeypatch.setattr(B.subprocess, "run", run)

    def compiled():
        calls.clear()
        B.build()
        return sorted(os.path.basename(c[c.index("-c") + 1]) for c in calls if "-c" in c)
    return files, compiled, calls


@pytest.mark.parametrize("what, again", [("a", ["a.cu"]), ("header", ["a.cu", "residual_norm.cu"]), ("abi", ["a.cu", "residual_norm.cu"]), ("build", ["a.cu", "residual_norm.cu"])])
def test_what_is_newer_is_compiled(tree, what, again):
    files, compiled, calls = tree
    assert compiled() == ["a.cu", "residual_norm.cu"]
    flags = {os.path.basename(c[c.index("-c") + 1]): c for c in calls if "-c" in c}
    assert "--use_fast_math" in flags["a.cu"] and "--use_fast_math" not in flags["residual_norm.cu"]
    assert compiled() == [] and not calls
    os.utime(files[what], (3000, 3000))
    assert compiled() == again and any("-shared" in c for c in calls)
