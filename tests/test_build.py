"""What the build makes where a part of its tools is missing; compilers and linkers are stood in for (no GPU, no nvcc)."""
import subprocess

import pytest
import torch  # noqa: F401  (imported before subprocess.run is replaced)

from dfdx_b200 import build


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
    for name in ("LIB", "MODULE"):
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    monkeypatch.setattr(build.subprocess, "run", t.run)
    return t


@pytest.mark.parametrize("why", ["fatal error: Python.h: No such file or directory", FileNotFoundError("g++")])
def test_the_library_is_made_without_the_python_module(tools, why):
    tools.failing["g++"] = why
    build.MODULE.write_text("of an earlier source")
    with pytest.warns(RuntimeWarning, match="was not built"):
        assert build.build(force=True) == build.LIB
    assert build.LIB.exists() and not build.MODULE.exists()


def test_a_failing_library_is_an_error(tools):
    tools.failing["nvcc"] = "error"
    with pytest.raises(RuntimeError, match="nvcc failed"):
        build.build(force=True)
    assert not build.LIB.exists()


def test_both_are_made_and_then_kept(tools):
    build.build()
    assert build.LIB.exists() and build.MODULE.exists()
    n = len(tools.commands)
    build.build()
    assert len(tools.commands) == n
