"""The build recipe in a directory of its own, with programs of this test's making in the compilers' place."""
import os
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stream-k.tvm_b200")

# a compiler: writes to what -o names (and, as a C++ compiler that is told to, fails)
COMPILER = """#!/bin/sh
echo "$0 $*" >> "{log}"
[ -n "$FAIL" ] && exit 1
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then echo made > "$2"; fi
  shift
done
"""

RUN = """
import importlib.util, os, sys
{before}
spec = importlib.util.spec_from_file_location("recipe", {recipe!r})
recipe = importlib.util.module_from_spec(spec)
spec.loader.exec_module(recipe)
for name in ("LIBDIR", "OBJDIR"):
    setattr(recipe, name, {tmp!r})
recipe.HOST_LIB = os.path.join({tmp!r}, os.path.basename(recipe.HOST_LIB))
{call}
"""

# torch cannot be imported, nor found
NO_TORCH = """
class Blocked:
    def find_spec(self, name, path=None, target=None):
        if name.split(".")[0] == "torch":
            raise ModuleNotFoundError("No module named 'torch'", name="torch")
sys.meta_path.insert(0, Blocked())
real = importlib.util.find_spec
importlib.util.find_spec = lambda name, package=None: None if name == "torch" else real(name, package)
"""


@pytest.fixture
def run(tmp_path):
    log = tmp_path / "log"
    for name in ("nvcc", "cxx"):
        path = tmp_path / name
        path.write_text(COMPILER.format(log=log))
        path.chmod(0o755)

    def go(call, before="", **env):
        code = RUN.format(before=before, recipe=os.path.join(PKG, "build.py"), tmp=str(tmp_path), call=call)
        r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=tmp_path, timeout=300,
                           env=dict({k: v for k, v in os.environ.items() if not k.startswith("STREAMK_")},
                                    NVCC=str(tmp_path / "nvcc"), CXX=str(tmp_path / "cxx"), **env))
        assert r.returncode == 0, r.stderr
        return r
    go.dir = tmp_path
    go.commands = lambda: log.read_text().splitlines() if log.exists() else []
    return go


def test_the_library_is_built_without_torch(run):
    run("assert os.path.exists(recipe.build())", before=NO_TORCH)
    assert (run.dir / "libstreamk_b200.so").exists()
    assert not [c for c in run.commands() if "sk_torch_host" in c]


def test_the_library_stands_if_the_host_module_does_not_compile(run):
    (run.dir / "cxx").write_text("#!/bin/sh\necho no compiler >&2\nexit 1\n")
    r = run("assert os.path.exists(recipe.build())")
    assert (run.dir / "libstreamk_b200.so").exists() and "sk_torch_host.cpp was not built" in r.stderr
    r = run("try: recipe.build_host()\nexcept RuntimeError as e: print('refused', e)")
    assert "refused" in r.stdout                  # asked for by name, it is an error


def test_both_are_built_with_torch(run):
    run("recipe.build()")
    assert (run.dir / "libstreamk_b200.so").exists()
    assert [f for f in os.listdir(run.dir) if f.startswith("sk_torch_host") and f.endswith(".so")]
    done = len(run.commands())
    run("recipe.build()")                         # nothing is stale
    assert len(run.commands()) == done
