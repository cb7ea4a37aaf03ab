"""Grouped products of small whole numbers, bit for bit.

Operands are whole numbers from -2 to 2, so every partial sum is a whole number below 2^24 and exact in
fp32 whatever its order; the result is the sum rounded once to its type, and a step of K that is left
out or counted twice where a sum is shared by several CTA pairs shows up, however long the sum is.
(A bound on rounding errors grows with the number of terms and lets such a step pass in long sums.)
"""
import pytest
import torch

import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"
RUN = {"nt": sk.streamk_grouped_nt, "nn": sk.streamk_grouped_nn, "tn": sk.streamk_grouped_tn}


def _whole(g, dtype, *shape):
    return torch.randint(-2, 3, shape, generator=g, device=DEV).to(dtype)


def _case(kind, sizes, N, K, dtype, lead=0, rest=0):
    T = lead + sum(sizes) + rest
    g = torch.Generator(device=DEV).manual_seed(T + N + K)
    A = _whole(g, dtype, T, K)
    B = _whole(g, dtype, T, N) if kind == "tn" else _whole(g, dtype, len(sizes), *((N, K) if kind == "nt" else (K, N)))
    off = torch.tensor([lead + sum(sizes[:i]) for i in range(len(sizes) + 1)], device=DEV)
    return A, B, off


def _sum(kind, A, B, off, skip=None):
    """In 64 bits; skip: 64 terms of every sum that are left out."""
    bounds = off.tolist()
    E = len(bounds) - 1
    a, b = A.double(), B.double()
    out = torch.zeros(*((E, A.shape[1], B.shape[1]) if kind == "tn" else (A.shape[0], B.shape[1 if kind == "nt" else 2])),
                      dtype=torch.float64, device=DEV)
    for e in range(E):
        lo, hi = bounds[e], bounds[e + 1]
        if kind == "tn":
            x, y = a[lo:hi].clone(), b[lo:hi]
            if skip is not None:
                x[skip * 64:skip * 64 + 64] = 0
            out[e] = x.T @ y
        else:
            x = a[lo:hi].clone()
            if skip is not None:
                x[:, skip * 64:skip * 64 + 64] = 0
            out[lo:hi] = x @ (b[e].T if kind == "nt" else b[e])
    return out


# Few tiles and long sums, which are shared by up to four pairs: K (TN: rows) in steps of 64 that the
# pairs divide unevenly, so that their runs begin inside tiles and reach into the next one; last
# steps of one term, of 16 and a few more, and whole ones.
SPLIT = [
    ("nt", [5], 256, 1600), ("nt", [1], 8, 20000), ("nt", [3, 0, 40], 300, 2504), ("nt", [17], 1000, 12808), ("nt", [300, 7], 520, 4104),
    ("nt", [64, 1, 1, 64], 264, 6472), ("nt", [33], 2000, 2200), ("nn", [16], 8, 20000), ("nn", [130, 0, 0, 9], 264, 8200),
    ("nn", [1, 31, 33], 776, 1608), ("nn", [250], 1032, 3336), ("nn", [5, 6, 7], 512, 9048), ("nn", [2], 4000, 1544),
    ("tn", [4001], 256, 256), ("tn", [3001, 0, 700], 264, 300), ("tn", [1025, 2049, 511, 17], 72, 520), ("tn", [9999], 40, 64),
    ("tn", [8209, 15000], 200, 136), ("tn", [6300], 1000, 500), ("tn", [2112, 4113, 0, 5000], 128, 128),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind,sizes,N,K", SPLIT)
def test_shared_sums(kind, sizes, N, K, dtype):
    A, B, off = _case(kind, sizes, N, K, dtype, lead=3, rest=2)
    ref = _sum(kind, A, B, off)
    assert float(ref.abs().max()) < 2 ** 16 - 32        # exact in fp32, finite in fp16
    steps = -(-(max(sizes) if kind == "tn" else K) // 64)
    for skip in (0, steps // 4, steps // 2, steps - 2):  # what this test has to notice, it does
        assert bool((_sum(kind, A, B, off, skip).to(dtype) != ref.to(dtype)).any()), skip
    for _ in range(3):
        assert torch.equal(RUN[kind](A, B, off), ref.to(dtype))
    assert torch.equal(RUN[kind](A, B, off, pdl=False), ref.to(dtype))
    if kind == "tn":
        assert torch.equal(sk.streamk_grouped_tn(A, B, off, out_dtype=torch.float32), ref.float())
    for num_sms in (10, 33):                             # other numbers of pairs, other runs
        assert torch.equal(RUN[kind](A, B, off, num_sms=num_sms), ref.to(dtype))
    sk.check_status()


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
@pytest.mark.parametrize("sizes,N,K", [([1000, 3, 0, 517], 520, 328), ([255, 256, 257, 1], 392, 1000), ([40] * 33, 264, 136),
                                       ([2300, 15, 31, 49], 1000, 520), ([16, 17, 32, 33, 48, 49, 64, 65], 776, 264)])
def test_whole_tiles(kind, sizes, N, K):
    A, B, off = _case(kind, sizes, N, K, torch.bfloat16, lead=1, rest=5)
    ref = _sum(kind, A, B, off)
    assert torch.equal(RUN[kind](A, B, off), ref.bfloat16())
    if kind == "tn":
        assert torch.equal(sk.streamk_grouped_tn(A, B, off, out_dtype=torch.float32), ref.float())
    sk.check_status()


def test_a_captured_layer_and_its_gradients():
    """The three products as a layer uses them, recorded once and replayed with other sizes."""
    E, N, K, T = 5, 264, 2504, 70
    A, W, off = _case("nt", [10, 0, 30, 1, 29], N, K, torch.float16)
    dY = _whole(torch.Generator(device=DEV).manual_seed(1), torch.float16, T, N)

    def run():
        return sk.streamk_grouped_nt(A, W, off), sk.streamk_grouped_nn(dY, W, off), sk.streamk_grouped_tn(dY, A, off)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for sizes in ([10, 0, 30, 1, 29], [70, 0, 0, 0, 0], [0, 0, 0, 0, 7], [14] * 5):
        off.copy_(torch.tensor([sum(sizes[:i]) for i in range(E + 1)]))
        graph.replay()
        for kind, r, a, b in zip(("nt", "nn", "tn"), got, (A, dY, dY), (W, W, A)):
            assert torch.equal(r, _sum(kind, a, b, off).half()), (kind, sizes)
        sk.check_status()
