"""Weight gradients in fp32 keep fp32's precision however many rows a group has.

The tensor cores truncate when they add, by less than a unit in the last place (2^-23 of the running
sum) for each of their instructions, which take 16 rows: a sum of n rows that they make alone is off by
up to n / 16 of those, all towards zero.  The kernel adds 512 rows at a time that way, 32 instructions,
and these sums in fp32, rounding to nearest (2^-24 each).  With independent rows a running sum is in the
norm never larger than its last value, and the parts' errors add up like the parts themselves, so the
whole is off by at most 32 x 2^-23 + n / 512 x 2^-24 of its norm.
"""
import pytest
import torch

import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,N,K", [([16384] * 8, 512, 512), ([100, 30000, 0, 513, 512], 776, 520), ([40000], 264, 256), ([60000, 3], 1000, 1032),
                                       ([8192] * 3, 77, 51)])
def test_error_in_the_norm(sizes, N, K, dtype):
    g = torch.Generator(device=DEV).manual_seed(N + K)
    A, B = (torch.randn(sum(sizes), n, generator=g, device=DEV).to(dtype) for n in (K, N))
    off = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], device=DEV)
    got = sk.streamk_grouped_tn(A, B, off, out_dtype=torch.float32)
    sk.check_status()
    for e, n in enumerate(sizes):
        if n == 0:
            assert not bool(got[e].any())
            continue
        rows = slice(sum(sizes[:e]), sum(sizes[:e]) + n)
        ref = A[rows].double().T @ B[rows].double()
        bound = min(32, -(-n // 16)) * 2.0 ** -23 + -(-n // 512) * 2.0 ** -24
        assert float((got[e].double() - ref).norm()) <= bound * float(ref.norm()), (e, n)
    assert torch.equal(sk.streamk_grouped_tn(A, B, off, out_dtype=torch.float32), got)


@pytest.mark.parametrize("rows", [1, 511, 512, 513, 1023, 1024, 1025, 1537, 5000])
@pytest.mark.parametrize("N,K,E", [(40, 64, 1), (300, 264, 3), (1000, 520, 20)])
def test_runs_of_whole_numbers(rows, N, K, E):
    """Every border between the runs, exactly: whole numbers, sums below 2^24."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    sizes = [rows, 0, 700, 3][:E] + [rows // 2] * max(0, E - 4)
    A, B = (torch.randint(-2, 3, (sum(sizes) + 2, n), generator=g, device=DEV).half() for n in (K, N))
    off = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], device=DEV)
    want = torch.stack([A[lo:hi].double().T @ B[lo:hi].double() for lo, hi in zip(off[:-1].tolist(), off[1:].tolist())])
    for num_sms in (None, 6):
        assert torch.equal(sk.streamk_grouped_tn(A, B, off, out_dtype=torch.float32, num_sms=num_sms), want.float())
    buf = torch.full((len(sizes), K, N + 5), 7.0, device=DEV)
    sk.streamk_grouped_tn(A, B, off, out=buf[..., :N], out_dtype=torch.float32)
    assert torch.equal(buf[..., :N], want.float()) and bool((buf[..., N:] == 7.0).all())
    sk.check_status()
