"""CPU checks of when the binding is built again (the compiler itself is replaced)."""
import os
import subprocess

import pytest
import torch

from scope_b200 import compile_lib


@pytest.fixture
def built(tmp_path, monkeypatch):
    """Counts the compilations; the outputs lie in a folder of their own."""
    monkeypatch.setattr(compile_lib, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(compile_lib, "BINDING", str(tmp_path / "_binding.so"))
    monkeypatch.setattr(compile_lib, "BINDING_STAMP", str(tmp_path / "_build" / "binding.stamp"), raising=False)
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(compile_lib.subprocess, "run", run)
    return calls


def test_the_binding_is_built_once(built):
    assert compile_lib.build_binding() == compile_lib.BINDING and os.path.exists(compile_lib.BINDING)
    compile_lib.build_binding()
    assert len(built) == 1
    compile_lib.build_binding(force=True)
    assert len(built) == 2


def test_another_pytorch_or_python_builds_it_again(built, monkeypatch):
    compile_lib.build_binding()
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    compile_lib.build_binding()
    assert len(built) == 2
    monkeypatch.setattr(compile_lib.sys, "version", "4.0")
    compile_lib.build_binding()
    assert len(built) == 3
    compile_lib.build_binding()
    assert len(built) == 3


def test_a_binding_without_a_stamp_is_built_again(built):
    compile_lib.build_binding()
    os.remove(compile_lib.BINDING_STAMP)
    compile_lib.build_binding()
    assert len(built) == 2
