"""The small-M kernel of the 8-bit integer product at every number of rows and of warps that its plan
can choose: the warps' sums meet where their rings were.  Exact sums, so the bits are known."""
import pytest
import torch

import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("N,K", [(32, 128), (40, 3000), (1000, 8192), (4736, 512), (4740, 2064), (8192, 4096), (9472, 1040), (9473, 200),
                                 (16384, 1024), (18944, 640), (20000, 272)])
@pytest.mark.parametrize("M", [1, 7, 8, 9, 15, 16])
def test_exact(M, N, K):
    g = torch.Generator(device=DEV).manual_seed(M * 31 + N + K)
    A = torch.randint(-128, 128, (M, K), generator=g, device=DEV, dtype=torch.int8)
    B = torch.randint(-128, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV) * 1e-3
    want = (((A.double() @ B.double().T).float() * sa[:, None]) * sb[None, :]).half()
    for _ in range(5):
        assert torch.equal(sk.streamk_int8_nt(A, B, sa, sb, schedule="gemv"), want)
    assert torch.equal(sk.streamk_int8_nt(A, B, sa, sb), want)
    sk.check_status()
