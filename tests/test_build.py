"""CPU tests of the in-tree build: the C library without torch, and when the torch binding is compiled again."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(cb):
    from cudaintro_b200 import build

    return build


@pytest.fixture
def compiled(build, monkeypatch, tmp_path):
    """The binding at a path of its own, not there yet, and a compiler that writes its command line there instead."""
    commands = []

    def compiler(cmd, **_):
        commands.append(cmd)
        with open(build.BINDING, "w") as f:
            f.write(" ".join(cmd))
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_torch_binding.so"))
    monkeypatch.setattr(build.subprocess, "run", compiler)
    return commands


def test_library_builds_without_torch(build, compiled, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # as on a machine that has none
    assert build.build() == build.LIB and os.path.exists(build.LIB)
    assert not compiled and not os.path.exists(build.BINDING)
    assert "torch" in capsys.readouterr().err


def test_library_builds_beside_a_torch_without_cuda(build, compiled, monkeypatch, capsys):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.version, "cuda", None)
    assert build.build() == build.LIB
    assert not compiled and "CUDA" in capsys.readouterr().err


def test_library_builds_without_the_headers_of_python(build, compiled, monkeypatch, capsys, tmp_path):
    pytest.importorskip("torch")
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert build.build() == build.LIB
    assert not compiled and "Python.h" in capsys.readouterr().err


def test_command_ends_well_without_torch(cb, tmp_path):
    """The documented command, in an interpreter whose torch cannot be imported, on a tree whose library is up to date."""
    pkg = tmp_path / "cudaintro_b200"
    shutil.copytree(os.path.join(ROOT, "cudaintro_b200"), pkg, ignore=shutil.ignore_patterns("_torch_binding.so", "build", "__pycache__"))
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    code = "import sys, runpy; sys.modules['torch'] = None; runpy.run_module('cudaintro_b200.build', run_name='__main__')"
    res = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    assert res.stdout.split()[-1] == str(pkg / "libb200gemm.so")
    assert not (pkg / "_torch_binding.so").exists()


def test_a_failing_compiler_is_an_error(build, compiled, monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **_: subprocess.CompletedProcess(cmd, 1, "", "no such thing"))
    with pytest.raises(RuntimeError, match="no such thing"):
        build.build()


def test_binding_is_compiled_again_for_another_torch_or_python(build, compiled, monkeypatch):
    """A binding that is newer than its source but was compiled for another torch or Python than those that ask for it."""
    pytest.importorskip("torch")
    from importlib import metadata

    build.build()
    assert len(compiled) == 1
    with open(build.BINDING, "ab") as f:  # what the compiler makes of the definition on its command line
        f.write(b"\0" + build.binding_target().encode() + b"\0")
    assert any(build.binding_target() in word for word in compiled[0])
    build.build()
    assert len(compiled) == 1  # up to date
    version, soabi = metadata.version, build.sysconfig.get_config_var
    monkeypatch.setattr(build.metadata, "version", lambda name: version(name) + ".post1")
    build.build()
    assert len(compiled) == 2 and any(version("torch") + ".post1" in word for word in compiled[1])
    monkeypatch.setattr(build.metadata, "version", version)
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399" if name == "SOABI" else soabi(name))
    build.build()
    assert len(compiled) == 3 and any("cpython-399" in word for word in compiled[2])


def test_built_binding_says_what_it_is_for(build):
    pytest.importorskip("torch")
    from cudaintro_b200 import capi

    assert callable(capi.linear_mxfp4)
    from cudaintro_b200 import _torch_binding

    assert _torch_binding.built_for == build.binding_target()
    assert build.binding_is_current()
