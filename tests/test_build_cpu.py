"""CPU: what the build of the Python module next to the library depends on.
Nothing is compiled: the compiler's command is recorded."""
import subprocess
from pathlib import Path

import pytest

from slm_turbo_b200 import build


@pytest.fixture
def tree(monkeypatch, tmp_path):
    """An up-to-date library, a module and its stamp in a folder of their own;
    the commands that a build runs."""
    monkeypatch.setattr(build, "_stale", lambda: False)
    monkeypatch.setattr(build, "HOST_PATH", tmp_path / "_host.so")
    monkeypatch.setattr(build, "HOST_STAMP", tmp_path / "_build" / "host.stamp")
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"module")
        return subprocess.CompletedProcess(cmd, 0)

    monkeypatch.setattr(build.subprocess, "run", run)
    return tmp_path, runs


def test_the_library_does_not_need_torch_or_a_cxx_compiler(tree, monkeypatch, capsys):
    tmp, runs = tree
    with monkeypatch.context() as m:
        m.setattr(build, "_torch_root", lambda: None)
        assert build.build_library() == build.LIB_PATH
    assert "torch" in capsys.readouterr().err
    with monkeypatch.context() as m:
        m.setattr(build, "_torch_root", lambda: tmp)  # a torch without CUDA
        assert build.build_library() == build.LIB_PATH
    assert "headers" in capsys.readouterr().err
    with monkeypatch.context() as m:
        real = build.shutil.which
        m.setattr(build.shutil, "which", lambda name: None if name == "g++" else real(name))
        assert build.build_library() == build.LIB_PATH
    assert "g++" in capsys.readouterr().err
    assert not runs and not build.HOST_PATH.exists()


def test_the_module_is_rebuilt_for_another_torch_or_python(tree, monkeypatch):
    _, runs = tree
    if build._host_tools()[1]:
        pytest.skip("no torch or C++ toolchain here")
    build.build_library()
    assert len(runs) == 1 and build.HOST_PATH.exists()
    build.build_library()
    assert len(runs) == 1  # up to date
    with monkeypatch.context() as m:
        m.setattr(build.importlib.metadata, "version", lambda name: "9.9.9")
        build.build_library()
        assert len(runs) == 2
        build.build_library()
        assert len(runs) == 2
    build.build_library()
    assert len(runs) == 3
    build.HOST_STAMP.unlink()  # of unknown origin
    build.build_library()
    assert len(runs) == 4


def test_toolkit_is_that_of_the_nvcc_in_use(tree, monkeypatch):
    """The compiler is the system's whatever $CXX says: the module shares the
    C++ runtime with torch."""
    tmp, runs = tree
    if build._host_tools()[1]:
        pytest.skip("no torch or C++ toolchain here")
    for d, f in (("toolkit/bin", "nvcc"), ("toolkit/include", "cuda_runtime_api.h"), ("cxx", "c++17")):
        (tmp / d).mkdir(parents=True)
        (tmp / d / f).write_text("")
        (tmp / d / f).chmod(0o755)
    monkeypatch.setenv("NVCC", str(tmp / "toolkit/bin/nvcc"))
    monkeypatch.setenv("CXX", str(tmp / "cxx/c++17"))
    build.build_library()
    assert Path(runs[0][0]).name == "g++" and str(tmp / "toolkit/include") in runs[0]
    assert "/usr/local/cuda/include" not in runs[0]
