"""The module of the decoding step is built for one PyTorch, and only that one loads it."""
import subprocess
import types

import pytest
import torch
import torch.utils.cpp_extension as ext

from oslo_b200.csrc import build
from oslo_b200.ops import _lib


def test_a_module_of_another_pytorch_is_not_loaded(monkeypatch):
    here = build.build_step()
    assert here == build.step_path() and here.exists()
    monkeypatch.setenv("OSLO_B200_AUTOBUILD", "0")
    assert _lib.step_calls.__wrapped__() is not None
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.step_path() != here and not build.step_path().exists()
    with pytest.warns(UserWarning, match="step module"):
        assert _lib.step_calls.__wrapped__() is None


def test_a_module_of_other_sources_is_not_loaded(monkeypatch, tmp_path):
    here = build.step_path()
    (tmp_path / "torch").mkdir()
    for name in ("torch/step_calls.cpp", "step_args.h"):
        (tmp_path / name).write_bytes((build.CSRC / name).read_bytes())
    monkeypatch.setattr(build, "CSRC", tmp_path)
    assert build.step_path() == here
    (tmp_path / "step_args.h").write_text("// other fields")
    assert build.step_path() != here


class _Compiler:
    """In place of subprocess.run: notes the command, and makes its output or fails."""

    def __init__(self, code):
        self.code, self.commands = code, []

    def __call__(self, cmd, **kw):
        self.commands.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        return types.SimpleNamespace(returncode=self.code, stdout="", stderr="no compiler")


def test_building_leaves_nothing_half_done(monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(build, "LIB_DIR", tmp_path)
    old = []  # include_paths before it took device types
    monkeypatch.setattr(ext, "include_paths", lambda cuda=False: old.append(cuda) or ["/headers"])
    fails = _Compiler(1)
    monkeypatch.setattr(subprocess, "run", fails)
    with pytest.raises(RuntimeError, match="no compiler"):
        build.build_step()
    assert old == [True] and "/headers" in fails.commands[0] and not list(tmp_path.iterdir())
    # the module is optional: what it does also goes through ctypes
    monkeypatch.setattr(build, "build_cuda", lambda verbose=False: "cuda")
    monkeypatch.setattr(build, "build_cpu", lambda: "cpu")
    assert build.build_all() == ("cuda", "cpu") and "no compiler" in capsys.readouterr().err
    works = _Compiler(0)
    monkeypatch.setattr(subprocess, "run", works)
    out = build.build_step()
    assert list(tmp_path.iterdir()) == [out] and works.commands[0][works.commands[0].index("-o") + 1] != str(out)
    assert build.build_step() == out and len(works.commands) == 1
