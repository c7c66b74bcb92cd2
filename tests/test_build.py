"""qwen4-thor_b200/build.py: what it starts, with the compilers replaced by records of their commands."""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(monkeypatch):
    spec = importlib.util.spec_from_file_location("q4t_build_under_test", os.path.join(ROOT, "qwen4-thor_b200", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.commands = []

    class Done:
        returncode = 0

        def __init__(self, cmd, **_):
            module.commands.append(cmd)

        def communicate(self):
            return "", None
    monkeypatch.setattr(subprocess, "Popen", Done)
    monkeypatch.setattr(subprocess, "run", lambda cmd, **_: Done(cmd))
    return module


def compiled(build):
    return [c for c in build.commands if "-c" in c]


def test_library_without_pytorch(build, monkeypatch, capsys):
    """A C or C++ user's build: every CUDA source, both libraries, no Python module."""
    monkeypatch.setitem(sys.modules, "torch", None)      # any import of it is an ImportError
    assert build.build(force=True) == build.LIB
    assert len(compiled(build)) == len(build.SOURCES) + len(build.CHECK_SOURCES)
    assert [c for c in build.commands if "-shared" in c and "-o" in c and c[c.index("-o") + 1] in (build.LIB, build.CHECK_LIB)]
    assert not any(build.CALLS in c for c in build.commands)
    assert "q4t_calls.so is left out" in capsys.readouterr().err


def test_python_module_with_pytorch(build):
    pytest.importorskip("torch")
    assert build.build(force=True) == build.LIB
    assert len(compiled(build)) == len(build.SOURCES) + len(build.CHECK_SOURCES)
    assert sum(build.CALLS in c for c in build.commands) == 1
