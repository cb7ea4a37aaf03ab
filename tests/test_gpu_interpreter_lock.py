"""The shortcut of the host path allocates and launches without the interpreter's lock, as a ctypes call
does: a launch that waits for room in the device's queue must not keep other Python threads from
running, since what the queue waits for may need one of them."""
import ctypes

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
