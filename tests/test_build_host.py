"""The build recipe without a compiler: what is built in which order, and what counts as up to date."""
import os
import subprocess

import pytest
import torch

from conftest import pkg


class Tools:
    """Stands in for nvcc and g++: writes what a command was to write, or fails where the first word is in `broken`."""

    def __init__(self, monkeypatch, build, tmp_path, broken=()):
        self.ran, self.broken = [], broken
        monkeypatch.setattr(build, "LIB_PATH", str(tmp_path / "lib.so"))
        monkeypatch.setattr(build, "PKG_DIR", str(tmp_path))
        monkeypatch.setattr(build, "ROOT_DIR", str(tmp_path))
        monkeypatch.setattr(build, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
        monkeypatch.setattr(subprocess, "run", self.run)
        monkeypatch.setattr(subprocess, "Popen", self.popen)

    def run(self, cmd, **_):
        name = os.path.basename(cmd[0])
        self.ran.append((name, os.path.basename(cmd[cmd.index("-o") + 1]).removesuffix(".tmp").removesuffix(".tmp.o")))
        if name in self.broken:
            return subprocess.CompletedProcess(cmd, 1, stdout="no such header")
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, stdout="")

    def popen(self, cmd, **_):
        done = self.run(cmd)
        done.communicate = lambda: (done.stdout, None)
        return done


def test_the_library_is_built_where_the_binding_cannot_be(monkeypatch, tmp_path):
    """The C library does not need torch's headers."""
    build = pkg("build")
    tools = Tools(monkeypatch, build, tmp_path, broken=("g++",))
    with pytest.raises(RuntimeError, match="g\\+\\+"):
        build.build_library()
    assert (tmp_path / "lib.so").exists() and ("nvcc", "lib.so") in tools.ran


def test_a_binding_of_another_torch_or_python_is_not_up_to_date(monkeypatch, tmp_path):
    build = pkg("build")
    tools = Tools(monkeypatch, build, tmp_path)
    build.build_library()
    built = [t for t in tools.ran if t[0] == "g++"]
    assert len(built) == 1
    build.build_library()
    assert [t for t in tools.ran if t[0] == "g++"] == built  # nothing is out of date
    monkeypatch.setattr(torch, "__version__", "99.1")
    build.build_library()
    assert len([t for t in tools.ran if t[0] == "g++"]) == 2


def test_a_binding_of_another_torch_is_not_loaded(monkeypatch):
    ops = pkg("ops")
    monkeypatch.setattr(torch, "__version__", "99.1")
    with pytest.raises(RuntimeError, match="build.py"):
        ops._load_native()
