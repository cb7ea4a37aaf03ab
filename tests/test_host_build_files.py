"""What the build recipe writes appears whole or not at all, under its own name."""
import os

import pytest

import streamk_b200  # noqa: F401
from streamk_b200 import build_recipe


@pytest.fixture
def compiler(monkeypatch, tmp_path):
    """Stands in for every compiler: notes what it is told to write, and fails half way on demand."""
    state = type("State", (), dict(fail=None, outs=[]))()

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        state.outs.append(out)
        with open(out, "w") as f:
            failed = state.fail is not None and state.fail in " ".join(cmd)
            f.write("half" if failed else "whole")
        return type("Result", (), dict(returncode=int(failed), stdout="", stderr=""))
    for name in ("LIBDIR", "OBJDIR"):
        monkeypatch.setattr(build_recipe, name, str(tmp_path))
    monkeypatch.setattr(build_recipe, "HOST_LIB", str(tmp_path / "sk_torch_host.so"))
    monkeypatch.setattr(build_recipe.subprocess, "run", run)
    monkeypatch.delenv("STREAMK_B200_TRACE", raising=False)
    return state


def test_files_are_named_when_they_are_whole(compiler, tmp_path):
    made = [build_recipe.build_library(), build_recipe.build_host()]
    finished = {str(tmp_path / p) for p in os.listdir(tmp_path)}
    assert set(made) <= finished and not finished & set(compiler.outs)      # (written elsewhere, then renamed)
    assert all((tmp_path / p).read_text() == "whole" for p in os.listdir(tmp_path))


@pytest.mark.parametrize("what", ["-shared", "sk_quant", "sk_torch_host"])
def test_a_failure_leaves_what_was_there(compiler, tmp_path, what):
    build_recipe.build_library()
    build_recipe.build_host()
    before = sorted(os.listdir(tmp_path))
    compiler.fail = what
    with pytest.raises(RuntimeError):
        (build_recipe.build_host if what == "sk_torch_host" else build_recipe.build_library)(force=True)
    assert sorted(os.listdir(tmp_path)) == before
    assert all((tmp_path / p).read_text() == "whole" for p in before)
