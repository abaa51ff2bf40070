"""The build of the compiled short way (_linear_call.so): it may fail without the library, and is tried again when what it is built from changes.
Compilers are stood in for: nothing is compiled here."""
import os
import subprocess

import pytest

from pixelbox_amd import build


class Compilers:
    """hipcc and the host compiler: each writes its output file, or fails"""

    def __init__(self):
        self.host_fails = None
        self.ran = []

    def __call__(self, cmd):
        name = "host" if any(a.endswith("_linear_call.so") for a in cmd) else "hipcc"
        self.ran.append(name)
        if name == "host" and self.host_fails:
            raise self.host_fails
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(name)


@pytest.fixture
def tree(tmp_path, monkeypatch):
    for name in ("LIB", "STAMP", "CALL_LIB", "CALL_STAMP"):
        monkeypatch.setattr(build, name, str(tmp_path / os.path.basename(getattr(build, name))))
    monkeypatch.setattr(build, "_hipcc", lambda: "/opt/rocm/bin/hipcc")
    monkeypatch.setattr(build, "_compile", lambda src, verbose: src)
    compilers = Compilers()
    monkeypatch.setattr(build.subprocess, "check_call", compilers)
    return compilers


def test_both_are_built_once(tree):
    assert build.needs_build()
    build.build()
    assert sorted(tree.ran) == ["hipcc", "host"] and os.path.exists(build.LIB) and os.path.exists(build.CALL_LIB) and not build.needs_build()
    build.build()
    assert len(tree.ran) == 2


@pytest.mark.parametrize("failure", [FileNotFoundError("no g++"), subprocess.CalledProcessError(1, "g++")])
def test_a_short_way_that_cannot_be_built_does_not_stop_the_library(tree, failure, capsys):
    build.build()
    tree.host_fails = failure
    tree.ran.clear()
    build.build(force=True)
    assert sorted(tree.ran) == ["hipcc", "host"] and os.path.exists(build.LIB)
    assert not os.path.exists(build.CALL_LIB)  # an older one is not left to be loaded
    assert "could not be built" in capsys.readouterr().err
    assert not build.needs_build()  # and it is not tried again and again
    build.build()
    assert len(tree.ran) == 2
    tree.host_fails = None
    build.build(force=True)
    assert os.path.exists(build.CALL_LIB) and not build.needs_build()


def test_without_torch_there_is_only_the_library(tree, monkeypatch):
    monkeypatch.setattr(build, "_torch_dir", lambda: None)
    build.build()
    assert tree.ran == ["hipcc"] and not build.needs_build() and not os.path.exists(build.CALL_LIB)


def test_a_missing_file_is_built_again(tree):
    build.build()
    tree.ran.clear()
    os.remove(build.CALL_LIB)
    assert build.needs_build()
    build.build()
    assert tree.ran == ["host"] and os.path.exists(build.CALL_LIB)
    os.remove(build.LIB)
    build.build()
    assert tree.ran == ["host", "hipcc"]


def test_another_torch_builds_it_again_and_nothing_else(tree, tmp_path, monkeypatch):
    other = tmp_path / "torch"
    other.mkdir()
    (other / "version.py").write_text("__version__ = '9.9.1+rocm8.1'\ndebug = False\n")
    build.build()
    monkeypatch.setattr(build, "_torch_dir", lambda: str(other))
    assert build.needs_build() and "9.9.1+rocm8.1" in build.call_tag()
    tree.ran.clear()
    build.build()
    assert tree.ran == ["host"] and not build.needs_build()


def test_a_module_built_for_another_torch_is_not_used():
    from pixelbox_amd import linear

    class Module:
        built_for = build.call_tag()

    assert linear._usable(Module) is Module  # what the build writes in is what the call looks for
    Module.built_for = "torch 1.0.0 cpython-39-x86_64-linux-gnu"
    with pytest.warns(UserWarning, match="built for torch 1.0.0"):
        assert linear._usable(Module) is False
    with pytest.warns(UserWarning, match="unknown"):
        assert linear._usable(object()) is False
