"""Products grouped by expert against their definition in 64 bits.

Tolerance, element by element: the result's own rounding, half a step (eps / 2 of the value, and
half of the smallest subnormal), and the accumulation: every product of two 16-bit numbers is
exact in fp32, the sum of n of them passes through at most n additions, each off by at most
2^-23 of what it adds up (fp32, truncation allowed for), so n 2^-23 sum |a b|.
"""
import numpy as np
import pytest
import torch

import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def _offsets(sizes, lead=0, dtype=torch.int32):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]) + lead, dtype=dtype, device=DEV)


def _operands(T, E, N, K, dtype, seed, kind):
    g = torch.Generator(device=DEV).manual_seed(seed)
    A = torch.randn(T, K, generator=g, device=DEV).to(dtype)
    if kind == "tn":
        return A, torch.randn(T, N, generator=g, device=DEV).to(dtype)
    shape = (E, N, K) if kind == "nt" else (E, K, N)
    return A, (torch.randn(*shape, generator=g, device=DEV) * 0.05).to(dtype)


def _check(got, terms, ref, n, dtype):
    info = torch.finfo(dtype)
    tol = ref.abs() * (info.eps / 2) + terms * (n * 2.0 ** -23) + info.smallest_normal * info.eps / 2
    bad = ~((got.double() - ref).abs() <= tol * 1.0001)
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - ref).abs().max()))


def _verify(kind, A, B, sizes, lead, got, dtype=None):
    """Every group's part of `got`, and zeros elsewhere (TN: for empty groups)."""
    dtype = dtype or A.dtype
    lo = lead
    for e, n in enumerate(sizes):
        hi = lo + n
        if kind == "tn":
            if n == 0:
                assert not bool(got[e].any()), e
            else:
                a, b = A[lo:hi].double(), B[lo:hi].double()
                _check(got[e], a.abs().T @ b.abs(), a.T @ b, n, dtype)
        elif n:
            w = B[e].double().T if kind == "nt" else B[e].double()
            a = A[lo:hi].double()
            _check(got[lo:hi], a.abs() @ w.abs(), a @ w, A.shape[1], dtype)
        lo = hi
    if kind != "tn":
        assert not bool(got[:lead].any()) and not bool(got[lo:].any())


RUN = {"nt": sk.streamk_grouped_nt, "nn": sk.streamk_grouped_nn, "tn": sk.streamk_grouped_tn}

CASES = [  # sizes, N, K, rows before the first group, rows after the last
    ([1], 8, 8, 0, 0),
    ([3], 256, 64, 0, 0),
    ([0, 5, 0, 16, 17], 264, 136, 0, 0),
    ([40, 0, 1, 33], 1000, 520, 3, 5),
    ([64, 64], 512, 128, 0, 0),
    ([255, 256, 257, 1, 0], 392, 200, 0, 1),
    ([300, 7, 513], 776, 320, 9, 100),
    ([0, 0, 0], 64, 64, 4, 4),
    ([1000, 3], 1024, 72, 0, 0),
    ([2300, 15, 31, 49], 520, 264, 0, 7),
]


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_definition(case, dtype, kind):
    sizes, N, K, lead, rest = CASES[case]
    T = lead + sum(sizes) + rest
    A, B = _operands(T, len(sizes), N, K, dtype, case, kind)
    got = RUN[kind](A, B, _offsets(sizes, lead))
    sk.check_status()
    assert got.dtype == dtype
    _verify(kind, A, B, sizes, lead, got)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [2, 5, 6, 9])
def test_weight_gradient_in_fp32(case, dtype):
    sizes, N, K, lead, rest = CASES[case]
    A, B = _operands(lead + sum(sizes) + rest, len(sizes), N, K, dtype, case, "tn")
    got = sk.streamk_grouped_tn(A, B, _offsets(sizes, lead, torch.int64), out_dtype=torch.float32)
    sk.check_status()
    assert got.dtype == torch.float32
    _verify("tn", A, B, sizes, lead, got, torch.float32)


@pytest.mark.parametrize("kind,sizes,N,K", [
    ("nt", [5], 256, 1536), ("nt", [5, 0, 40], 300, 2504), ("nt", [300, 7], 520, 4096), ("nn", [130, 0, 0, 9], 264, 8192),
    ("nn", [16], 8, 20000), ("nn", [1, 31, 33], 776, 1600), ("nt", [1000], 256, 1536),
    ("tn", [4000], 256, 256), ("tn", [3001, 0, 700], 264, 300), ("tn", [1025, 2049, 511, 17], 72, 520), ("tn", [9999], 40, 64)])
def test_sums_split_over_pairs(kind, sizes, N, K):
    """Few tiles and long sums: several CTA pairs share a tile; twice the same bits."""
    A, B = _operands(sum(sizes), len(sizes), N, K, torch.bfloat16, N + K, kind)
    off = _offsets(sizes)
    got = RUN[kind](A, B, off)
    sk.check_status()
    _verify(kind, A, B, sizes, 0, got)
    for _ in range(5):
        assert torch.equal(RUN[kind](A, B, off), got)
    if kind == "tn":
        _verify(kind, A, B, sizes, 0, RUN[kind](A, B, off, out_dtype=torch.float32), torch.float32)


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
@pytest.mark.parametrize("E", [32, 33, 300, 1024])
def test_many_groups(E, kind):
    rng = np.random.default_rng(E)
    sizes = rng.integers(0, 6, E).tolist()
    sizes[E // 2] = 90
    sizes[-1] = 0
    N, K = (72, 64) if E > 100 else (264, 128)
    A, B = _operands(sum(sizes) + 3, E, N, K, torch.bfloat16, E, kind)
    got = RUN[kind](A, B, _offsets(sizes))
    sk.check_status()
    _verify(kind, A, B, sizes, 0, got)


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
def test_odd_extents_and_strides(kind):
    sizes = [10, 0, 70, 21]
    T = sum(sizes)
    for N, K in ((77, 51), (129, 100), (100, 129)):
        A, B = _operands(T, len(sizes), N, K, torch.float16, N, kind)
        _verify(kind, A, B, sizes, 0, RUN[kind](A, B, _offsets(sizes)))
    N, K = 200, 136
    A, B = _operands(T, len(sizes), N, K, torch.float16, 7, kind)
    want = RUN[kind](A, B, _offsets(sizes))
    Aw = torch.full((T, K + 40), NAN, dtype=torch.float16, device=DEV)
    Aw[:, 8:8 + K] = A
    Bw = torch.full((*B.shape[:-1], B.shape[-1] + 24), NAN, dtype=torch.float16, device=DEV)
    Bw[..., 16:16 + B.shape[-1]] = B
    got = RUN[kind](Aw[:, 8:8 + K], Bw[..., 16:16 + B.shape[-1]], _offsets(sizes))
    assert torch.equal(got, want)                     # (no NaN from beside the operands)
    if kind != "tn":                                   # every other expert of a larger set
        B2 = torch.full((2 * len(sizes), *B.shape[1:]), NAN, dtype=torch.float16, device=DEV)
        B2[::2] = B
        assert torch.equal(RUN[kind](A, B2[::2], _offsets(sizes)), want)
    At = A.t().contiguous().t()
    assert torch.equal(RUN[kind](At, B, _offsets(sizes)), want)


@pytest.mark.parametrize("kind", ["nt", "nn"])
def test_out_keeps_rows_of_no_group(kind):
    sizes, lead, rest, N, K = [30, 2, 0, 300], 5, 60, 136, 64
    T = lead + sum(sizes) + rest
    A, B = _operands(T, len(sizes), N, K, torch.bfloat16, 1, kind)
    want = RUN[kind](A, B, _offsets(sizes, lead))
    for pitch, first in ((N, 0), (N + 1, 0), (N + 8, 8), (N + 3, 1)):
        buf = torch.full((T, pitch + first), 3.0, dtype=torch.bfloat16, device=DEV)
        out = buf[:, first:first + N]
        assert RUN[kind](A, B, _offsets(sizes, lead), out=out) is out
        sk.check_status()
        assert torch.equal(out[lead:T - rest], want[lead:T - rest])
        buf[lead:T - rest, first:first + N] = 3.0
        assert bool((buf == 3.0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_weight_gradient_into_out(dtype):
    sizes, N, K = [30, 0, 300], 104, 72
    A, B = _operands(sum(sizes), 3, N, K, torch.float16, 1, "tn")
    want = sk.streamk_grouped_tn(A, B, _offsets(sizes), out_dtype=dtype)
    for extra_n, extra_k, first in ((0, 0, 0), (16, 3, 8), (5, 1, 3)):
        buf = torch.full((3, K + extra_k, N + extra_n + first), 3.0, dtype=dtype, device=DEV)
        out = buf[:, :K, first:first + N]
        sk.streamk_grouped_tn(A, B, _offsets(sizes), out=out, out_dtype=dtype)
        sk.check_status()
        assert torch.equal(out, want)
        out.fill_(3.0)
        assert bool((buf == 3.0).all())


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
@pytest.mark.parametrize("value", [NAN, float("inf"), float("-inf")])
def test_what_other_rows_hold_stays_there(kind, value):
    """Rows of no group hold NaN or infinities, and so does one group: the others do not see it."""
    sizes, lead, rest, N, K = [37, 50, 1, 63, 200], 7, 70, 264, 200
    T = lead + sum(sizes) + rest
    A, B = _operands(T, len(sizes), N, K, torch.bfloat16, 3, kind)
    off = _offsets(sizes, lead)
    want = RUN[kind](A, B, off)
    A2, B2 = A.clone(), B.clone()
    for t in (A2, B2) if kind == "tn" else (A2,):
        t[:lead] = value
        t[T - rest:] = value
        t[lead + 37:lead + 87] = value          # group 1
    got = RUN[kind](A2, B2, off)
    sk.check_status()
    if kind == "tn":
        keep = [0, 2, 3, 4]
        assert torch.equal(got[keep], want[keep])
        assert bool((~got[1].isfinite()).all())
    else:
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[lead + 37:lead + 87] = False
        assert torch.equal(got[keep], want[keep])
        assert bool((~got[~keep].isfinite()).all())
    if kind != "tn":                             # a group's own weights stay with it too
        B2 = B.clone()
        B2[3] = value
        got = RUN[kind](A, B2, off)
        assert torch.equal(got[:lead + 88], want[:lead + 88]) and torch.equal(got[lead + 151:], want[lead + 151:])


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
def test_offsets_out_of_order_are_clamped_and_reported(kind):
    T, E, N, K = 100, 4, 72, 64
    A, B = _operands(T, E, N, K, torch.float16, 5, kind)
    for bad, clamped in (([0, 50, 20, 80, 100], [0, 50, 50, 80, 100]), ([-5, 10, 200, 40, 400], [0, 10, 100, 100, 100]),
                         ([0, 2 ** 40, -2 ** 40, 7, 99], [0, 100, 100, 100, 100])):
        got = RUN[kind](A, B, torch.tensor(bad, dtype=torch.int64, device=DEV))
        with pytest.raises(sk.StreamKError):
            sk.check_status()
        want = RUN[kind](A, B, torch.tensor(clamped, dtype=torch.int64, device=DEV))
        sk.check_status()
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
def test_captured_and_replayed_with_other_sizes(kind):
    T, E, N, K = 260, 5, 264, 192
    A, B = _operands(T, E, N, K, torch.bfloat16, 5, kind)
    off = _offsets([100, 0, 60, 40, 60])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        RUN[kind](A, B, off)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        first = RUN[kind](A, B, off, pdl=True)
        second = RUN[kind](A, B, off, pdl=True)
    for sizes in ([0, 0, 0, 0, 0], [260, 0, 0, 0, 0], [17, 100, 3, 99, 41], [52] * 5):
        off.copy_(_offsets(sizes))
        g.replay()
        torch.cuda.synchronize()
        _verify(kind, A, B, sizes, 0, first)
        assert torch.equal(first, second)


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
def test_the_fast_path_and_the_long_one_agree(kind):
    sizes = [9, 0, 30]
    A, B = _operands(45, 3, 136, 200, torch.bfloat16, 2, kind)
    for off in (_offsets(sizes, 2), _offsets(sizes, 2, torch.int64)):
        want = RUN[kind](A, B, off)
        assert torch.equal(RUN[kind](A, B, off, pdl=False), want)
        assert torch.equal(RUN[kind](torch.nn.Parameter(A), torch.nn.Parameter(B), off), want)
        out = torch.zeros_like(want)
        assert torch.equal(RUN[kind](A, B, off, out=out), want)
    if kind == "tn":
        f32 = sk.streamk_grouped_tn(A, B, off, out_dtype=torch.float32)
        assert torch.equal(sk.streamk_grouped_tn(A, B, off, out_dtype=torch.float32, pdl=False), f32)


def test_two_streams_at_once():
    sizes = [100, 0, 260, 40]
    A, B = _operands(400, 4, 520, 256, torch.float16, 5, "nt")
    A2 = A.flip(0).contiguous()
    off = _offsets(sizes)
    want, want2 = sk.streamk_grouped_nt(A, B, off), sk.streamk_grouped_nt(A2, B, off)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(8):
        with torch.cuda.stream(streams[i & 1]):
            outs.append(sk.streamk_grouped_nt(A2 if i & 1 else A, B, off))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want2 if i & 1 else want)


def test_two_captured_graphs_replayed_at_once():
    """Graphs captured on one stream and replayed on two: each has a workspace of its own (the sums
    here are split, so the counters and the parts in it matter)."""
    g = torch.Generator(device=DEV).manual_seed(11)
    cases = []
    for i, (sizes, N, K) in enumerate((([5, 40], 300, 6400), ([130], 264, 8192))):
        A, B = _operands(sum(sizes), len(sizes), N, K, torch.bfloat16, i, "nt")
        q = torch.randint(-127, 128, (7, 8192), generator=g, device=DEV, dtype=torch.int8)
        w = torch.randint(-127, 128, (512, 8192), generator=g, device=DEV, dtype=torch.int8)
        s, t = torch.rand(7, generator=g, device=DEV), torch.rand(512, generator=g, device=DEV)
        run = lambda A=A, B=B, off=_offsets(sizes), q=q, w=w, s=s, t=t: [
            sk.streamk_grouped_nt(A, B, off), sk.streamk_int8_nt(q, w, s, t), sk.streamk_grouped_nt(A, B, off)]
        want = [r.clone() for r in run()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        cases.append((graph, got, want, run))        # (run holds the operands that the graph reads)
    sk.check_status()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for _, got, _, _ in cases:
            for r in got:
                r.fill_(7.0)
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _ in cases:
            for r, x in zip(got, want):
                assert torch.equal(r, x)


def test_branches_of_one_captured_graph():
    """Two streams recorded into one graph: their split sums run at the same time in every replay."""
    sizes, N, K = [5, 40], 300, 6400
    off = _offsets(sizes)
    pairs = [_operands(sum(sizes), len(sizes), N, K, torch.bfloat16, i, "nt") for i in range(2)]
    want = [sk.streamk_grouped_nt(A, B, off).clone() for A, B in pairs]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        got = [[], []]
        for _ in range(4):
            got[0].append(sk.streamk_grouped_nt(*pairs[0], off))
            with torch.cuda.stream(side):
                got[1].append(sk.streamk_grouped_nt(*pairs[1], off))
        main.wait_stream(side)
    for _ in range(10):
        for r in got[0] + got[1]:
            r.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for branch, x in zip(got, want):
            for r in branch:
                assert torch.equal(r, x)
    sk.check_status()


def _random(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(sum(shape)))


@pytest.mark.parametrize("kind", ["nt", "nn"])
def test_addresses_beyond_32_bits(kind):
    """More than 2^31 elements in the rows, in the weights and in the result: what lies behind them
    is right."""
    for T, E, N, K in ((600_000, 3, 136, 4096), (70_000, 2, 33_000, 72), (40, 70, 8192, 4096)):
        A = _random(T, K)
        B = _random(E, N, K) if kind == "nt" else _random(E, K, N)
        last = 37 if T > 100 else 3
        sizes = [0] * E
        sizes[0], sizes[-1] = T - last, last
        got = RUN[kind](A, B, _offsets(sizes))
        _verify(kind, A[-last:], B[-1:], [last], 0, got[-last:])
        a = A[:5].clone()
        _verify(kind, a, B, [5] + [0] * (E - 1), 0, got[:5])
        sk.check_status()


def test_weight_gradient_beyond_32_bits():
    A, B = _random(600_000, 4096), _random(600_000, 72)         # rows of a group behind 2^31 elements
    got = sk.streamk_grouped_tn(A, B, _offsets([599_900, 0, 100]))
    _verify("tn", A[-100:], B[-100:], [100], 0, got[2:])
    assert not bool(got[1].any())
    A, B = _random(300, 8192), _random(300, 4096)               # a result of 2^31 elements and more
    sizes = [0] * 66
    sizes[0], sizes[-2] = 100, 200
    for N in (4096, 4095):
        got = sk.streamk_grouped_tn(A, B[:, :N], _offsets(sizes), out_dtype=torch.float32)
        _verify("tn", A[100:], B[100:, :N], [200], 0, got[-2:-1])
        assert not bool(got[-1].any()) and not bool(got[1:-2].any())
        del got
    sk.check_status()


def test_few_sms():
    sizes = [100, 0, 260, 40]
    for kind in ("nt", "nn", "tn"):
        A, B = _operands(400, 4, 520, 256, torch.float16, 5, kind)
        want = RUN[kind](A, B, _offsets(sizes))
        for n in (2, 3, 10):
            got = RUN[kind](A, B, _offsets(sizes), num_sms=n)
            sk.check_status()
            _verify(kind, A, B, sizes, 0, got)
        assert torch.equal(RUN[kind](A, B, _offsets(sizes)), want)


def test_gradients_against_differences():
    """<dY, Y(X + h U) - Y(X - h U)> / 2h = <dX, U>, and the same for W: the product is linear in
    each, so with operands that are small whole numbers everything is exact but the gradients'
    own rounding, and there is none in fp16 below 2048."""
    g = torch.Generator(device=DEV).manual_seed(0)
    sizes, N, K = [5, 0, 20, 9], 40, 24
    E, T = len(sizes), sum(sizes)

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=g, device=DEV).half()

    X, W, dY, U, V, off = whole(T, K), whole(E, N, K), whole(T, N), whole(T, K), whole(E, N, K), _offsets(sizes)
    dX, dW = sk.streamk_grouped_nn(dY, W, off), sk.streamk_grouped_tn(dY, X, off)
    y = [sk.streamk_grouped_nt(a, w, off).double() for a, w in ((X + U, W), (X - U, W), (X, W + V), (X, W - V))]
    assert float((dY.double() * (y[0] - y[1])).sum()) / 2 == float((dX.double() * U.double()).sum())
    assert float((dY.double() * (y[2] - y[3])).sum()) / 2 == float((dW.double() * V.double()).sum())


def test_no_rows():
    off = torch.zeros(4, dtype=torch.int32, device=DEV)
    A, W = torch.empty(0, 64, dtype=torch.half, device=DEV), torch.randn(3, 40, 64, device=DEV).half()
    assert sk.streamk_grouped_nt(A, W, off).shape == (0, 40)
    dW = sk.streamk_grouped_tn(A, torch.empty(0, 16, dtype=torch.half, device=DEV), off)
    assert dW.shape == (3, 64, 16) and not bool(dW.any())


def test_refusals():
    A, B = _operands(20, 3, 40, 64, torch.float16, 1, "nt")
    off = _offsets([5, 5, 10])
    for bad, err in (((A.cpu(), B, off), ValueError), ((A, B.cpu(), off), ValueError), ((A, B, off.cpu()), ValueError),
                     ((A.float(), B.float(), off), TypeError), ((A, B.bfloat16(), off), TypeError),
                     ((A, B, off.float()), TypeError), ((A, B, off[:-1]), ValueError), ((A, B, off[None]), ValueError),
                     ((A, B, off[:1]), ValueError), ((A, B[:, :, :32], off), ValueError), ((A, B[0], off), ValueError),
                     ((A[0], B, off), ValueError), ((A, B[:, :0], off), ValueError)):
        with pytest.raises(err):
            sk.streamk_grouped_nt(*bad)
    with pytest.raises(ValueError):
        sk.streamk_grouped_nn(A, B, off)                        # B is [E,N,K], K does not match
    with pytest.raises(ValueError):
        sk.streamk_grouped_tn(A, A[:10], off)
    with pytest.raises(TypeError):
        sk.streamk_grouped_tn(A, A, off, out_dtype=torch.bfloat16)
    for out in (torch.empty(20, 41, dtype=torch.half, device=DEV), torch.empty(20, 40, dtype=torch.bfloat16, device=DEV),
                torch.empty(40, 20, dtype=torch.half, device=DEV).t(), torch.empty(1, 40, dtype=torch.half, device=DEV).expand(20, 40)):
        with pytest.raises(ValueError):
            sk.streamk_grouped_nt(A, B, off, out=out)
    with pytest.raises(sk.StreamKError):
        sk.streamk_grouped_nt(A, B, off, num_sms=1)             # CTA pairs
    with pytest.raises(sk.StreamKError):
        big = torch.zeros(1025, 8, 8, dtype=torch.half, device=DEV)
        sk.streamk_grouped_nt(A[:, :8], big, torch.zeros(1026, dtype=torch.int32, device=DEV))


def test_a_layer_of_experts_with_a_quantised_shared_expert():
    """The operators as a model's feed-forward layer uses them: routed experts (grouped up and down
    products over rows sorted by expert) beside a dense expert in 8 bits."""
    g = torch.Generator(device=DEV).manual_seed(8)
    tokens, top, E, D, H = 45, 2, 6, 256, 384
    x = torch.randn(tokens, D, generator=g, device=DEV).half()
    up, down = ((torch.randn(*s, generator=g, device=DEV) * 0.06).half() for s in ((E, H, D), (E, D, H)))
    up_s, down_s = ((torch.randn(*s, generator=g, device=DEV) * 0.06).half() for s in ((H, D), (D, H)))
    gate = torch.randn(tokens, E, generator=g, device=DEV)
    weight, expert = gate.softmax(-1).topk(top)
    order = expert.flatten().argsort(stable=True)
    counts = torch.bincount(expert.flatten(), minlength=E)
    off = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
    rows = x[order // top]
    h = torch.relu(sk.streamk_grouped_nt(rows, up, off))
    y = sk.streamk_grouped_nt(h, down, off)
    routed = torch.zeros(tokens, D, device=DEV).index_add_(0, order // top, y.float() * weight.flatten()[order][:, None])
    q, s = sk.int8_quantize(x)
    hs = torch.relu(sk.streamk_int8_nt(q, *_weight(up_s, s)))
    q2, s2 = sk.int8_quantize(hs)
    shared = sk.streamk_int8_nt(q2, *_weight(down_s, s2))
    sk.check_status()
    # the same in 64 bits
    xd = x.double()
    ref = torch.zeros(tokens, D, dtype=torch.float64, device=DEV)
    for e in range(E):
        for k in range(top):
            m = expert[:, k] == e
            ref[m] += weight[m, k].double()[:, None] * (torch.relu(xd[m] @ up[e].double().T) @ down[e].double().T)
    # two fp16 roundings (of h and y, 2^-11 each, h's carried through a sum of H terms) and fp32 sums
    assert float((routed.double() - ref).abs().max()) <= 2e-3 * float(ref.abs().max())
    refs = torch.relu(xd @ up_s.double().T) @ down_s.double().T
    assert float((shared.double() - refs).norm()) <= 3e-2 * float(refs.norm())


def _weight(w, sx):
    """The 8-bit form of a weight and both scales, in the order that streamk_int8_nt takes them."""
    q, s = sk.int8_quantize(w)
    return q, sx, s
