"""When the build compiles the extension of the dense operators again, and what it leaves when that fails; the compiler's place is taken."""
import os
import types

import pytest
import torch


@pytest.fixture
def build(monkeypatch, tmp_path):
    """The build with its outputs in another place and a compiler that makes empty files."""
    from haste_b200 import build as b
    calls = []

    def run(cmd, **_):
        calls.append(cmd)
        fails = getattr(b, "compiler_fails", lambda c: False)(cmd)
        if not fails:
            open(cmd[cmd.index("-o") + 1], "w").close()
        return types.SimpleNamespace(returncode=int(fails), stdout="", stderr="no such header")

    monkeypatch.setattr(b, "OBJ", str(tmp_path / "build"))
    monkeypatch.setattr(b, "DENSE", str(tmp_path / "_dense.so"))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b.subprocess, "run", run)
    os.makedirs(b.OBJ)
    return b, calls


def test_another_torch_is_noticed(build, monkeypatch):
    b, calls = build
    for _ in range(2):
        b._build_dense(False)
        assert len(calls) == 1                                              # made once, then up to date
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    for _ in range(2):
        b._build_dense(False)
        assert len(calls) == 2
    b._build_dense(True)
    assert len(calls) == 3


def test_the_library_is_there_where_the_extension_fails(build, monkeypatch):
    b, calls = build
    monkeypatch.setattr(b, "compiler_fails", lambda cmd: "dense_binding.cpp" in " ".join(cmd), raising=False)
    with pytest.raises(RuntimeError, match="dense_binding.cpp failed"):
        b.build()
    assert os.path.exists(b.LIB) and not os.path.exists(b.DENSE)
