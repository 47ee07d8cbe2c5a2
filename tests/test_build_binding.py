"""CPU: when the Python binding is compiled again (the compiler is a fake)."""

from __future__ import annotations

import subprocess
from types import SimpleNamespace

import torch

from nova_b200 import build


def test_rebuilt_for_another_torch(monkeypatch, tmp_path):
    runs = []

    def compiler(cmd, **kw):
        runs.append(cmd)
        build.FAST.write_bytes(b"")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build, "FAST", tmp_path / "_fast.so")
    monkeypatch.setattr(build, "OBJ", tmp_path)
    monkeypatch.setattr(subprocess, "run", compiler)
    build.build_binding()
    build.build_binding()
    assert len(runs) == 1                                     # up to date
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    build.build_binding()
    build.build_binding()
    assert len(runs) == 2
    build.build_binding(force=True)
    assert len(runs) == 3
