"""The shortcut module of the host path is a convenience: without it the entry points go the longer way."""
import warnings

import pytest
import torch

import streamk_b200 as sk
from streamk_b200 import _lib as L
from streamk_b200 import ops


@pytest.fixture(params=[ImportError("undefined symbol"), OSError("not found"), RuntimeError("compiling failed")],
                ids=lambda e: type(e).__name__)
def broken(request, monkeypatch):
    def fail():
        raise request.param
    monkeypatch.setattr(L, "load_host", fail)
    monkeypatch.setattr(ops, "_fast", None)


def _calls():
    h, q = torch.zeros(4, 32, dtype=torch.half), torch.zeros(4, 32, dtype=torch.int8)
    s, off = torch.ones(4), torch.tensor([0, 4])
    return [lambda: sk.int8_quantize(h), lambda: sk.streamk_int8_nt(q, q, s, s), lambda: sk.streamk_grouped_nt(h, h[None], off),
            lambda: sk.streamk_grouped_nn(h, h[None], off), lambda: sk.streamk_grouped_tn(h, h, off)]


@pytest.mark.parametrize("i", range(5))
def test_calls_go_the_longer_way_and_say_so_once(broken, i):
    with pytest.warns(RuntimeWarning, match="longer host path"):
        with pytest.raises(ValueError, match="no CPU path"):      # (what that way says to CPU tensors)
            _calls()[i]()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for call in _calls():
            with pytest.raises(ValueError, match="no CPU path"):
                call()


@pytest.mark.gpu
def test_results_without_the_shortcut(monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(0)
    X = torch.randn(50, 256, generator=g, device="cuda").half()
    W = torch.randn(3, 40, 256, generator=g, device="cuda").half()
    off = torch.tensor([0, 10, 10, 50], device="cuda")

    def run():
        q, s = sk.int8_quantize(X)
        return [q, s, sk.streamk_int8_nt(q, q, s, s), sk.streamk_grouped_nt(X, W, off),
                sk.streamk_grouped_nn(X[:, :40].contiguous(), W, off), sk.streamk_grouped_tn(X[:, :40].contiguous(), X, off)]
    want = run()

    def fail():
        raise OSError("not found")
    with monkeypatch.context() as m:
        m.setattr(L, "load_host", fail)
        m.setattr(ops, "_fast", None)
        with pytest.warns(RuntimeWarning):
            got = run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            replayed = run()
        graph.replay()
        again = run()
        sk.check_status()
        for results in (got, replayed, again):
            for a, b in zip(results, want):
                assert torch.equal(a, b)
    monkeypatch.setattr(ops, "_fast", None)                       # (registers the workspaces afresh)
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


def test_a_missing_kernel_library_is_still_an_error(monkeypatch, tmp_path):
    monkeypatch.setattr(L, "_lib", None)
    monkeypatch.setattr(L, "_host", None)
    monkeypatch.setattr(ops, "_fast", None)
    monkeypatch.setenv("STREAMK_B200_LIB", str(tmp_path / "absent.so"))
    with pytest.raises(OSError):
        sk.int8_quantize(torch.zeros(4, 32, dtype=torch.half))
