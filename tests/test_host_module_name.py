"""The host module belongs to the torch and the Python that it was compiled against."""
import os
import sys

import torch

import streamk_b200  # noqa: F401
from streamk_b200 import build_recipe


def test_the_name_tells_the_versions(monkeypatch):
    path = build_recipe.host_lib()
    name = os.path.basename(path)
    assert os.path.dirname(path) == build_recipe.LIBDIR and name.startswith("sk_torch_host.") and name.endswith(".so")
    assert torch.__version__ in name and sys.implementation.cache_tag in name
    monkeypatch.setattr(torch, "__version__", "9.9.9+x/y")
    other = os.path.basename(build_recipe.host_lib())
    assert other != name and "/" not in other


def test_another_torch_does_not_take_the_old_module(monkeypatch, tmp_path):
    made = []

    def compile_(cmd, **kw):
        made.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("made")
        return type("Result", (), dict(returncode=0, stdout="", stderr=""))
    monkeypatch.setattr(build_recipe, "LIBDIR", str(tmp_path))
    monkeypatch.setattr(build_recipe, "HOST_LIB", str(tmp_path / "sk_torch_host.so"))
    monkeypatch.setattr(build_recipe.subprocess, "run", compile_)
    first = build_recipe.build_host()
    assert build_recipe.build_host() == first and len(made) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    second = build_recipe.build_host()
    assert second != first and len(made) == 2 and os.path.exists(first) and os.path.exists(second)


def test_what_is_loaded_is_that_file():
    from streamk_b200 import _lib as L
    assert os.path.samefile(L.load_host().__file__, build_recipe.host_lib())
