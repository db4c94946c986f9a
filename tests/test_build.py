"""What the build makes where a part of its tools is missing; compilers and linkers are stood in for (no GPU, no nvcc)."""
import subprocess

import pytest
import torch

from dfdx_b200 import build, heads


@pytest.fixture
def tools(tmp_path, monkeypatch):
    """A build into tmp_path: commands are recorded and make the file behind -o, or fail as `tools.failing` says."""
    class Tools:
        def __init__(self):
            self.commands, self.failing = [], {}

        def run(self, cmd, **kwargs):
            self.commands.append(cmd)
            tool = cmd[0].rsplit("/", 1)[-1]
            if isinstance(self.failing.get(tool), Exception):
                raise self.failing[tool]
            if tool in self.failing:
                return subprocess.CompletedProcess(cmd, 1, "", self.failing[tool])
            open(cmd[cmd.index("-o") + 1], "w").write(tool)
            return subprocess.CompletedProcess(cmd, 0, "", "")

    t = Tools()
    monkeypatch.setattr(build, "LIBDIR", tmp_path)
    monkeypatch.setattr(build, "OBJDIR", tmp_path / "obj")
    monkeypatch.setattr(build, "LIB", tmp_path / build.LIB.name)
    monkeypatch.setattr(build.subprocess, "run", t.run)
    return t


@pytest.mark.parametrize("why", ["fatal error: Python.h: No such file or directory", FileNotFoundError("g++")])
def test_the_library_is_made_without_the_python_module(tools, why):
    tools.failing["g++"] = why
    build.module_path().write_text("of an earlier source")
    with pytest.warns(RuntimeWarning, match="was not built"):
        assert build.build(force=True) == build.LIB
    assert build.LIB.exists() and not build.module_path().exists()


def test_a_failing_library_is_an_error(tools):
    tools.failing["nvcc"] = "error"
    with pytest.raises(RuntimeError, match="nvcc failed"):
        build.build(force=True)
    assert not build.LIB.exists()


def test_both_are_made_and_then_kept(tools):
    build.build()
    assert build.LIB.exists() and build.module_path().exists()
    n = len(tools.commands)
    build.build()
    assert len(tools.commands) == n


def test_a_module_of_another_torch_is_neither_kept_nor_loaded(tools, monkeypatch):
    build.build()
    before, n = build.module_path(), len(tools.commands)
    monkeypatch.setattr(heads, "_module", None)
    monkeypatch.setattr(torch, "__version__", "99.0.1")
    assert build.module_path() != before
    with pytest.raises(RuntimeError, match="is missing"):
        heads._host()
    build.build()
    assert [c[0] for c in tools.commands[n:]] == ["g++"] and build.module_path().exists() and before.exists()


def test_the_module_is_named_after_the_python(monkeypatch):
    before = build.module_path()
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: ".cpython-399.so")
    assert build.module_path() != before and build.module_path().name.endswith(".cpython-399.so")
