"""CPU: the native calls are compiled again for another torch or Python, and only then."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("qik_build", ROOT / "qwen-image-kernel_b200" / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    monkeypatch.setattr(b, "CALLS", tmp_path / "_calls.so")
    monkeypatch.setattr(b, "OBJ", tmp_path / "obj")
    monkeypatch.setattr(b, "CALLS_MADE_FOR", tmp_path / "obj" / "_calls.made_for", raising=False)
    ran = []

    def compiler(cmd, check):
        ran.append(cmd)
        b.CALLS.write_text("")
    monkeypatch.setattr(b.subprocess, "run", compiler)
    b.ran = ran
    return b


def test_calls_are_made_again_for_another_torch(build, monkeypatch):
    build.build_calls()
    build.build_calls()
    assert len(build.ran) == 1
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "9.9.9")
        build.build_calls()
        build.build_calls()
        assert len(build.ran) == 2
    build.build_calls()
    assert len(build.ran) == 3
    with monkeypatch.context() as m:
        m.setattr(build.sys, "version", "3.99")
        build.build_calls()
    assert len(build.ran) == 4
    build.build_calls(force=True)
    assert len(build.ran) == 5
    src = build.CSRC / "calls.cpp"
    os.utime(build.CALLS, (0, src.stat().st_mtime - 10))
    build.build_calls()
    assert len(build.ran) == 6


def test_a_failed_compile_is_tried_again(build, monkeypatch):
    build.build_calls()
    with monkeypatch.context() as m:
        m.setattr(build.subprocess, "run", lambda *a, **k: (_ for _ in ()).throw(RuntimeError("no")))
        with pytest.raises(RuntimeError):
            build.build_calls(force=True)
    build.build_calls()
    assert len(build.ran) == 2
