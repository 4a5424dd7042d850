"""The in-tree build (CPU): the library does not wait for the serving calls, which are a Python module over torch."""
from __future__ import annotations

import ctypes
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """pyrite_b200.build with its outputs under tmp_path and one host source in the library."""
    from pyrite_b200 import build
    monkeypatch.setattr(build, "SOURCES", ["quantize.cpp"])
    monkeypatch.setattr(build, "OBJ", tmp_path / "obj")
    monkeypatch.setattr(build, "LIB", tmp_path / "libpyrite_b200.so")
    return build


NO_TORCH = """
import sys
from pathlib import Path
sys.modules["torch"] = None  # import torch raises
out = Path(sys.argv[1])
from pyrite_b200 import build
build.SOURCES, build.OBJ, build.LIB = ["quantize.cpp"], out / "obj", out / "libpyrite_b200.so"
assert build.build() == build.LIB
import pyrite_b200.kernels.native
"""


def test_library_builds_without_torch(tmp_path):
    run = subprocess.run([sys.executable, "-c", NO_TORCH, str(tmp_path)], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    assert "serving calls" in run.stderr and "torch" in run.stderr  # what is missing is said
    assert ctypes.CDLL(str(tmp_path / "libpyrite_b200.so")).pyrite_quantize_types(None, 0) > 0


def test_library_is_linked_when_the_serving_calls_fail(tree, monkeypatch):
    def broken(force=False):
        raise RuntimeError("g++ failed for serving_calls.cpp")

    monkeypatch.setattr(tree, "build_calls", broken)
    with pytest.warns(RuntimeWarning, match="serving calls.*g\\+\\+ failed"):
        assert tree.build() == tree.LIB
    assert tree.LIB.is_file()


def test_serving_calls_of_other_sources_are_not_loaded(tmp_path, monkeypatch):
    """The module's file name follows its source and the C interface: one built from others is not found."""
    from pyrite_b200 import build
    for name in ("csrc/serving_calls.cpp", "include/pyrite_b200.h"):
        (tmp_path / name).parent.mkdir(parents=True, exist_ok=True)
    (tmp_path / "csrc/serving_calls.cpp").write_bytes((build.CSRC / "serving_calls.cpp").read_bytes())
    (tmp_path / "include/pyrite_b200.h").write_bytes((ROOT / "include" / "pyrite_b200.h").read_bytes())
    here = build.calls_path()
    monkeypatch.setattr(build, "CSRC", tmp_path / "csrc")
    monkeypatch.setattr(build, "ROOT", tmp_path)
    assert build.calls_path() == here
    names = {here}
    for name in ("csrc/serving_calls.cpp", "include/pyrite_b200.h"):
        with open(tmp_path / name, "a") as f:
            f.write("// changed\n")
        names.add(build.calls_path())
    assert len(names) == 3


def test_builds_at_once_write_files_of_their_own(tree, monkeypatch, tmp_path):
    """Two builds at once, of an object, the serving calls and the library: no file is written by both, none is left
    behind."""
    import threading
    real, wrote, both = subprocess.run, [], threading.Barrier(2, timeout=60)
    monkeypatch.setattr(tree, "calls_path", lambda: tmp_path / "serving_calls.so")

    def run(cmd, **kw):
        if "-o" in cmd:  # both builds are here before either writes
            wrote.append(cmd[cmd.index("-o") + 1])
            both.wait()
            Path(wrote[-1]).write_bytes(b"x")
            return subprocess.CompletedProcess(cmd, 0, "", "")
        return real(cmd, **kw)

    monkeypatch.setattr(tree.subprocess, "run", run)
    for job, out in ((lambda: tree.build_calls(force=True), tmp_path / "serving_calls.so"),
                     (lambda: tree.link([]), tree.LIB),
                     (lambda: tree._compile(Path("a.cu"), tmp_path / "a.o", False) or tmp_path / "a.o",
                      tmp_path / "a.o")):
        wrote.clear()
        with ThreadPoolExecutor(2) as pool:
            assert {f.result() for f in [pool.submit(job) for _ in range(2)]} == {out}
        assert len(set(wrote)) == 2 and out.is_file()
    assert sorted(p.name for p in tmp_path.iterdir()) == ["a.o", "libpyrite_b200.so", "serving_calls.so"]
