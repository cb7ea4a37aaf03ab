"""Errors that a replayed kernel reports reach check_status(), although the workspace that a captured
call works in belongs to its graph and is zeroed at the start of every replay."""
import pytest
import torch

import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _offsets(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
def test_offsets_out_of_order_in_a_replay(kind):
    run = {"nt": sk.streamk_grouped_nt, "nn": sk.streamk_grouped_nn, "tn": sk.streamk_grouped_tn}[kind]
    A = torch.randn(100, 64, device=DEV).half()
    B = torch.randn(100, 72, device=DEV).half() if kind == "tn" else torch.randn(4, *((72, 64) if kind == "nt" else (64, 72)), device=DEV).half()
    good, bad = _offsets([0, 20, 50, 80, 100]), _offsets([0, 50, 20, 80, 100])
    off = good.clone()
    want = run(A, B, good).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(A, B, off)
    graph.replay()
    sk.check_status()
    off.copy_(bad)
    for _ in range(3):                      # (the first error stays through the replays that follow)
        graph.replay()
    off.copy_(good)
    graph.replay()
    with pytest.raises(sk.StreamKError, match="captured") as e:
        sk.check_status()
    assert e.value.status == 8              # SK_ERR_ARG
    sk.check_status()                       # reported once
    assert torch.equal(got, want)
    off.copy_(bad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):           # replayed on another stream than the one that asks
        graph.replay()
    side.synchronize()
    with pytest.raises(sk.StreamKError):
        sk.check_status()
    graph.replay()
    torch.cuda.synchronize()
    del graph, got                          # the graph and its memory are gone, the report is not
    run(A, B, good, pdl=False)
    with pytest.raises(sk.StreamKError):
        sk.check_status()
    run(A, B, good)
    sk.check_status()


def test_errors_of_eager_calls_stay_with_their_stream():
    A, B = torch.randn(100, 64, device=DEV).half(), torch.randn(4, 72, 64, device=DEV).half()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sk.streamk_grouped_nt(A, B, _offsets([0, 50, 20, 80, 100]))
    side.synchronize()
    sk.check_status()
    with torch.cuda.stream(side):
        with pytest.raises(sk.StreamKError, match="device status"):
            sk.check_status()
        sk.check_status()


def test_a_wait_that_runs_out_in_a_replay():
    """Two CTAs share a tile and one is told not to publish its flag: the other gives up after its
    limit and reports."""
    g = torch.Generator(device=DEV).manual_seed(1)
    A, B = (torch.randint(-127, 128, (128, 2048), generator=g, device=DEV, dtype=torch.int8) for _ in range(2))
    sa, sb = torch.rand(128, device=DEV), torch.rand(128, device=DEV)
    kw = dict(schedule="streamk", tile_m=128, tile_n=128, num_sms=2)
    want = sk.streamk_int8_nt(A, B, sa, sb, **kw).clone()
    graphs = []
    for drop in (None, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sk.streamk_int8_nt(A, B, sa, sb, timeout_us=20000, _drop_flag_cta=drop, **kw)
        graphs.append((graph, out))
    graphs[0][0].replay()
    sk.check_status()
    graphs[1][0].replay()
    with pytest.raises(sk.StreamKError, match="captured") as e:
        sk.check_status()
    assert e.value.status == 6              # SK_ERR_FIXUP_TIMEOUT
    graphs[0][0].replay()
    sk.check_status()
    assert torch.equal(graphs[0][1], want)
