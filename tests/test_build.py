"""CPU tests of the build: which compiler is needed for what, and what a build leaves alone."""
import os
import sysconfig

import pytest

from dfssm_b200 import _lib, build


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """The commands that a build into an empty folder would run."""
    ran = []
    monkeypatch.setattr(build, "LIBDIR", str(tmp_path / "lib"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib" / "libdfssm.so"))
    monkeypatch.setattr(build, "PYCALLS", str(tmp_path / "lib" / os.path.basename(build.PYCALLS)))

    def run(cmd, **_):
        ran.append(os.path.basename(cmd[0]))
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.delenv("CXX", raising=False)
    monkeypatch.setattr(build, "nvcc", lambda: "nvcc")
    return ran


def test_library_comes_first(commands):
    assert build.build() == build.LIB and os.path.exists(build.LIB) and os.path.exists(build.PYCALLS)
    assert commands == ["nvcc", "g++"]
    build.build()
    assert commands == ["nvcc", "g++"]  # nothing is stale


def test_library_without_pythons_headers(commands, monkeypatch, tmp_path, capsys):
    """The C library needs nvcc alone; the module is left out, and said to be."""
    paths = {**sysconfig.get_paths(), "include": str(tmp_path)}
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: paths)
    assert build.build() == build.LIB and commands == ["nvcc"] and not os.path.exists(build.PYCALLS)
    assert "Python.h" in capsys.readouterr().err


def test_module_is_this_pythons():
    """The module's name holds the interpreter's ABI: another Python builds its own."""
    assert _lib.PYCALLS_PATH == build.PYCALLS
    assert build.PYCALLS.endswith("dfssm_pycalls" + sysconfig.get_config_var("EXT_SUFFIX"))


def test_calls_without_the_module_say_so(monkeypatch, tmp_path):
    pytest.importorskip("torch")
    monkeypatch.setattr(_lib, "_pycalls", None)
    monkeypatch.setattr(_lib, "PYCALLS_PATH", str(tmp_path / "none.so"))
    with pytest.raises(RuntimeError, match="dfssm_b200.build"):
        _lib.pycalls()
