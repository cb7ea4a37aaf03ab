"""The workspace of a captured call is let go by the next call outside a capture, whichever way that
call takes to the library."""
import pytest
import torch

import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _int8():
    q, s = torch.ones(40, 256, dtype=torch.int8, device=DEV), torch.ones(40, device=DEV)
    return lambda: sk.streamk_int8_nt(q, q, s, s)


def _grouped():
    A, B = torch.ones(30, 64, device=DEV).half(), torch.ones(2, 40, 64, device=DEV).half()
    off = torch.tensor([0, 10, 30], device=DEV)
    return lambda: sk.streamk_grouped_nt(A, B, off)


@pytest.mark.parametrize("make", [_int8, _grouped])
def test_a_plain_eager_call_lets_go_of_it(make):
    run = make()
    want = run().clone()
    before = sk.cached_memory_bytes()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        held = sk.cached_memory_bytes()
        assert held > before                          # for the calls of the same capture that may follow
        assert torch.equal(run(), want)               # a plain call: nothing to copy, no options
        assert sk.cached_memory_bytes() == before
        assert torch.equal(run(), want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del graph, out
    sk.check_status()


def test_the_memory_goes_with_the_graph():
    run = _int8()
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    del graph
    run()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    base = torch.cuda.memory_reserved()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    del graph
    run()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    assert torch.cuda.memory_reserved() <= base


def test_calls_of_one_capture_share_one():
    run = _int8()
    run()
    before = sk.cached_memory_bytes()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
        one = sk.cached_memory_bytes()
        run()
        assert sk.cached_memory_bytes() == one > before
    run()
    assert sk.cached_memory_bytes() == before
