"""The shortcut of the host path allocates and launches without the interpreter's lock, as a ctypes call
does: a launch that waits for room in the device's queue must not keep other Python threads from
running, since what the queue waits for may need one of them."""
import ctypes
import threading

import pytest
import torch

import streamk_b200 as sk
from streamk_b200 import _lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def module():
    """The shortcut, bound to a function that launches nothing and returns whether its thread holds
    the lock (1, which reads as a refusal, or 0, which reads as success)."""
    X = torch.ones(8, 64, device=DEV, dtype=torch.half)
    q, s, off = torch.ones(8, 64, device=DEV, dtype=torch.int8), torch.ones(8, device=DEV), torch.tensor([0, 8], device=DEV)
    sk.streamk_int8_nt(q, q, s, s)                       # (the stream has its workspace)
    lib, m = L.load(), L.load_host()
    held = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p).value
    m.bind(held, held, held)
    yield m, X, q, s, off
    m.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (lib.sk_quantize_i8, lib.sk_gemm_i8, lib.sk_gemm_grouped)))


def test_the_lock_is_let_go(module):
    m, X, q, s, off = module
    assert m.quantize(X) is not None
    assert m.gemm_i8(q, q, s, s, False) is not None
    for kind, B in ((0, X[None]), (1, X.t().contiguous()[None]), (2, X)):
        assert m.grouped(kind, X, B, off, False) is not None, kind
    assert ctypes.pythonapi.PyGILState_Check() == 1      # and taken back


def test_an_allocation_that_fails_takes_it_back(module):
    m, X, q, s, off = module
    A = torch.ones(1, 65536, device=DEV, dtype=torch.half)
    offsets = torch.zeros(1024, device=DEV, dtype=torch.int64)
    assert m.grouped(2, A, A, offsets, False) is None    # 8 TB: refused, left to the longer path ...
    assert ctypes.pythonapi.PyGILState_Check() == 1
    with pytest.raises(torch.OutOfMemoryError):          # ... which says why
        sk.streamk_grouped_tn(A, A, offsets)


@pytest.mark.parametrize("own_stream", [True, False])
def test_calls_from_several_threads(own_stream):
    """Each thread with a stream of its own, or all on one."""
    g = torch.Generator(device=DEV).manual_seed(3)
    sizes, N, K = [5, 40, 0, 200], 300, 3336                # (short ones: shared sums in the workspace)
    A = torch.randint(-2, 3, (sum(sizes), K), generator=g, device=DEV).half()
    W = torch.randint(-2, 3, (len(sizes), N, K), generator=g, device=DEV).half()
    q = torch.randint(-127, 128, (7, 8192), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(-127, 128, (512, 8192), generator=g, device=DEV, dtype=torch.int8)
    sa, sb = torch.rand(7, generator=g, device=DEV), torch.rand(512, generator=g, device=DEV)
    off = torch.tensor([0, 5, 45, 45, 245], device=DEV)

    def run():
        return [sk.streamk_grouped_nt(A, W, off), sk.streamk_int8_nt(q, w, sa, sb), *sk.int8_quantize(A),
                sk.streamk_grouped_tn(A[:, :256], A[:, :128], off)]
    want = [r.clone() for r in run()]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(4)

    def work(stream):
        with torch.cuda.stream(stream):
            start.wait()
            for _ in range(50):
                got = run()
                stream.synchronize()
                wrong.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))
    one = torch.cuda.Stream()
    threads = [threading.Thread(target=work, args=(torch.cuda.Stream() if own_stream else one,)) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    sk.check_status()
