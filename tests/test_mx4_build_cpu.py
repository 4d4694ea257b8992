"""How the MX4 binding is found and built (no GPU needed)."""
import os
import subprocess
import types

import torch

from _int4 import build, cuda_loader, mx4


def test_binding_belongs_to_its_source_and_to_torch(monkeypatch, tmp_path):
    """Another source or another torch is another file: a build that does not fit is never loaded."""
    here = build.binding_path()
    assert build.binding_path() == here and os.path.dirname(here) == os.path.dirname(build.lib_path())
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.binding_path() != here
    monkeypatch.undo()
    for name in ("mx4_binding.cpp", "convrot_b200.h"):
        src = [p for p in build.binding_sources() if p.endswith(name)]
        assert len(src) == 1
        changed = tmp_path / name
        changed.write_bytes(open(src[0], "rb").read() + b"\n")
        monkeypatch.setattr(build, "binding_sources", lambda p=src[0], c=str(changed), all=build.binding_sources(): [c if q == p else q for q in all])
        assert build.binding_path() != here
        monkeypatch.undo()


def test_builds_of_two_processes_do_not_share_a_temporary_file(monkeypatch, tmp_path):
    seen = []

    def run(cmd, **_):
        out = cmd[cmd.index("-o") + 1]
        seen.append(out)
        open(out, "wb").close()
        return types.SimpleNamespace(returncode=0, stderr="", stdout="")
    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(build, "lib_path", lambda: str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "binding_path", lambda: str(tmp_path / "_mx4_binding_x.so"))
    for pid in (11, 12):
        monkeypatch.setattr(os, "getpid", lambda p=pid: p)
        build.build()
        build.build_binding()
    assert len(set(seen)) == 4
    assert sorted(os.listdir(tmp_path)) == ["_mx4_binding_x.so", "lib.so"]


def test_native_loads_the_library_through_its_own_loader(monkeypatch):
    """One lock for the library's build, whoever asks first."""
    called = []
    monkeypatch.setattr(mx4, "_native", None)
    monkeypatch.setattr(cuda_loader, "library", lambda: called.append(1))
    mx4.native()
    assert called
