"""When the torch binding is built, and when it is left alone (no compiler runs here)."""
import os

import pytest

from nim_lowprec_b200 import build as B

torch = pytest.importorskip("torch")


@pytest.fixture
def calls(tmp_path, monkeypatch):
    """The build with its results in a folder of their own and a compiler that only writes
    them; the commands that it was given."""
    lib = tmp_path / "liblowprec_cuda.so"
    lib.write_bytes(b"")
    os.utime(lib, (1, 1))
    monkeypatch.setattr(B, "OUT", str(lib))
    monkeypatch.setattr(B, "OBJDIR", str(tmp_path))
    monkeypatch.setattr(B, "BINDING", str(tmp_path / "_torch_binding.so"))
    got = []

    def run(cmd, check):
        got.append(cmd)
        open(cmd[cmd.index("-o") + 1], "wb").close()
    monkeypatch.setattr(B.subprocess, "run", run)
    return got


def test_built_once(calls):
    B.build_binding()
    assert len(calls) == 1
    B.build_binding()
    assert len(calls) == 1
    B.build_binding(force=True)
    assert len(calls) == 2


def test_a_torch_without_cuda_is_left_out(calls, monkeypatch, capsys):
    monkeypatch.setattr(torch.version, "cuda", None)
    B.build_binding()
    B.build_binding(force=True)
    assert not calls
    said = capsys.readouterr().out.splitlines()
    assert len(said) == 2 and all("without CUDA" in s for s in said)


@pytest.mark.parametrize("what", ["torch", "python"])
def test_another_torch_or_python_makes_it_stale(calls, monkeypatch, what):
    B.build_binding()
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    else:
        monkeypatch.setattr(B.sys, "version", "9.9.9")
    B.build_binding()
    assert len(calls) == 2
    B.build_binding()
    assert len(calls) == 2
