"""8-bit integer product and its quantiser against their definitions.

The sums are integers, so the product has one right answer: the exact sum rounded to fp32, times
scale_a, times scale_b (a rounding each), rounded to 16 bits.  Every schedule is compared bit for
bit.  The quantiser's codes are compared with the exact quotient's nearest integers (rational
arithmetic where it matters), its scales with the correctly rounded ones.
"""
import fractions

import pytest
import torch

import oracle
import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(M, N, K, seed, low=-128):
    g = torch.Generator().manual_seed(seed)
    A = torch.randint(low, 128, (M, K), generator=g, dtype=torch.int8)
    B = torch.randint(low, 128, (N, K), generator=g, dtype=torch.int8)
    sa = torch.rand(M, generator=g) * 0.01 + 1e-4
    sb = torch.rand(N, generator=g) * 0.01 + 1e-4
    return A, B, sa, sb


def _ref(A, B, sa, sb, dtype):
    total = A.double() @ B.double().T          # exact: below 2^53
    return ((total.float() * sa[:, None]) * sb[None, :]).to(dtype)


def _bits(t):
    return t.cpu().view(torch.int16)


SHAPES = [(100, 500, 5000), (70, 1900, 6200), (1, 1, 1), (1, 128, 128), (1, 1000, 333), (2, 300, 1024), (7, 11008, 512), (16, 512, 4096), (17, 129, 640), (33, 4096, 1024),
          (64, 384, 8192), (65, 640, 2048), (100, 1000, 1000), (128, 1024, 1040), (250, 1536, 1024), (384, 384, 8192),
          (513, 1030, 257), (1024, 2048, 512), (2049, 4104, 384), (4096, 4096, 256)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product_is_exact_under_every_schedule(shape, dtype):
    A, B, sa, sb = _case(*shape, seed=sum(shape))
    ref = _bits(_ref(A, B, sa, sb, dtype))
    d = [t.to(DEV) for t in (A, B, sa, sb)]
    for schedule in ("auto", "streamk", "hybrid", "hybrid_dp_first", "dp"):
        C = sk.streamk_int8_nt(*d, out_dtype=dtype, schedule=schedule)
        sk.check_status()
        assert torch.equal(_bits(C), ref), schedule
    try:
        fits = sk.schedule_info(*shape, kind="int8", schedule="cluster")["cluster"] > 0
    except sk.StreamKError:
        fits = False
    if fits:
        C = sk.streamk_int8_nt(*d, out_dtype=dtype, schedule="cluster")
        sk.check_status()
        assert torch.equal(_bits(C), ref)


@pytest.mark.parametrize("tiles", [(256, 256), (256, 96), (256, 32), (128, 256), (128, 128), (128, 80), (16, 128), (48, 128), (16, 40)])
@pytest.mark.parametrize("shape", [(40, 520, 1056), (300, 777, 656)], ids=lambda s: "x".join(map(str, s)))
def test_tiles(shape, tiles):
    A, B, sa, sb = _case(*shape, seed=tiles[0] + tiles[1])
    ref = _bits(_ref(A, B, sa, sb, torch.float16))
    for schedule in ("streamk", "dp", "hybrid"):
        C = sk.streamk_int8_nt(A.to(DEV), B.to(DEV), sa.to(DEV), sb.to(DEV), schedule=schedule, tile_m=tiles[0],
                               tile_n=tiles[1])
        sk.check_status()
        assert torch.equal(_bits(C), ref), schedule


@pytest.mark.parametrize("shape", [(300, 2048, 512), (4200, 4000, 200)], ids=lambda s: "x".join(map(str, s)))
def test_strides_out_and_unaligned_operands(shape):
    M, N, K = shape
    A, B, sa, sb = _case(M, N, K, seed=5)
    ref = _bits(_ref(A, B, sa, sb, torch.float16))
    Aw = torch.zeros(M, K + 48, dtype=torch.int8, device=DEV)
    Aw[:, 16:16 + K] = A.to(DEV)
    Bw = torch.zeros(N, K + 7, dtype=torch.int8, device=DEV)       # rows that TMA cannot address: copied
    Bw[:, 3:3 + K] = B.to(DEV)
    out = torch.full((M, N + 3), 7.0, dtype=torch.float16, device=DEV)
    C = sk.streamk_int8_nt(Aw[:, 16:16 + K], Bw[:, 3:3 + K], sa.to(DEV)[:, None], sb.to(DEV)[None, :], out=out[:, :N])
    sk.check_status()
    assert C.data_ptr() == out.data_ptr()
    assert torch.equal(_bits(out[:, :N].contiguous()), ref)
    assert bool((out[:, N:] == 7.0).all())
    At = A.t().contiguous().to(DEV).t()                             # column-major: copied
    assert torch.equal(_bits(sk.streamk_int8_nt(At, B.to(DEV), sa.to(DEV), sb.to(DEV))), ref)


def test_largest_sum_and_the_limit_of_k():
    K = 131071
    A = torch.full((3, K), -128, dtype=torch.int8)
    B = torch.full((20, K), -128, dtype=torch.int8)
    B[1] = 127
    sa = torch.tensor([1e-6, 2e-6, 0.0])
    sb = torch.full((20,), 1e-3)
    ref = _bits(_ref(A, B, sa, sb, torch.float16))
    for schedule in ("auto", "streamk", "cluster"):
        C = sk.streamk_int8_nt(A.to(DEV), B.to(DEV), sa.to(DEV), sb.to(DEV), schedule=schedule)
        sk.check_status()
        assert torch.equal(_bits(C), ref), schedule
    with pytest.raises(sk.StreamKError):
        sk.streamk_int8_nt(torch.zeros(1, K + 1, dtype=torch.int8, device=DEV),
                           torch.zeros(16, K + 1, dtype=torch.int8, device=DEV), sa[:1].to(DEV), sb[:16].to(DEV))


def test_scales_that_are_not_finite_or_tiny():
    A, B, sa, sb = _case(20, 200, 256, seed=9)
    sa[3], sa[4], sb[7], sb[8] = float("nan"), float("inf"), 0.0, 1e-30
    ref = _ref(A, B, sa, sb, torch.float16)
    C = sk.streamk_int8_nt(A.to(DEV), B.to(DEV), sa.to(DEV), sb.to(DEV)).cpu()
    assert torch.equal(C.isnan(), ref.isnan())
    assert torch.equal(C.nan_to_num(1.0), ref.nan_to_num(1.0))


def test_two_streams_and_a_captured_graph():
    A, B, sa, sb = (t.to(DEV) for t in _case(256, 1024, 2048, seed=3))
    A2 = A.flip(0).contiguous()
    want, want2 = _bits(sk.streamk_int8_nt(A, B, sa, sb)), _bits(sk.streamk_int8_nt(A2, B, sa, sb))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i & 1]):
            outs.append(sk.streamk_int8_nt(A2 if i & 1 else A, B, sa, sb))
    torch.cuda.synchronize()
    for i, c in enumerate(outs):
        assert torch.equal(_bits(c), want2 if i & 1 else want)
    X = torch.randn(256, 2048, device=DEV, dtype=torch.float16)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q, sx = sk.int8_quantize(X)
        out = sk.streamk_int8_nt(q, B, sx, sb)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        q, sx = sk.int8_quantize(X)
        out = sk.streamk_int8_nt(q, B, sx, sb, pdl=True)
    X.copy_(torch.randn(256, 2048, device=DEV, dtype=torch.float16))
    g.replay()
    torch.cuda.synchronize()
    q1, s1 = sk.int8_quantize(X)
    assert torch.equal(_bits(out), _bits(sk.streamk_int8_nt(q1, B, s1, sb)))


def test_the_fast_path_and_the_long_one_agree():
    """Plain calls take a shortcut from tensors to the C ABI; options, copies and refusals do not."""
    A, B, sa, sb = (t.to(DEV) for t in _case(70, 264, 512, seed=2))
    want = _bits(_ref(*(t.cpu() for t in (A, B, sa, sb)), torch.float16))
    for kw in ({}, {"pdl": False}, {"schedule": "dp"}, {"num_sms": 20}):
        assert torch.equal(_bits(sk.streamk_int8_nt(A, B, sa, sb, **kw)), want), kw
    P = torch.nn.Parameter(torch.randn(33, 512, device=DEV).half())     # a parameter is a plain tensor
    for x in (P, P.detach()[::2], P.detach()[:, 16:272]):
        (q, s), (q2, s2) = sk.int8_quantize(x), sk.int8_quantize(x, pdl=False)
        assert torch.equal(q, q2) and torch.equal(s, s2) and not q.requires_grad and not s.requires_grad
    held = sk.cached_memory_bytes()
    assert held > 0
    sk.release_cached_memory()                                          # the shortcut lets go of it, too
    assert sk.cached_memory_bytes() == 0
    assert torch.equal(_bits(sk.streamk_int8_nt(A, B, sa, sb)), want)
    assert sk.cached_memory_bytes() > 0


# ------------------------------------------------------------------------------------ quantiser
def _codes(x):
    """Nearest integers (halves to even) of 127 x / a in exact rational arithmetic; x: 1-D."""
    v = [fractions.Fraction(float(t)) for t in x]
    a = max(abs(t) for t in v)
    return [round(127 * t / a) if a else 0 for t in v]     # round() of a Fraction: halves to even


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 100), (16, 1024), (2, 1032), (4, 4096), (3, 4100), (2, 11008),
                                   (1, 12296), (2, 32768), (1, 40000), (130, 257), (1000, 64)],
                         ids=lambda s: "x".join(map(str, s)))
def test_codes_and_scales(shape, dtype):
    M, K = shape
    g = torch.Generator().manual_seed(M * 7 + K)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    q, s = sk.int8_quantize(x.to(DEV))
    assert q.dtype == torch.int8 and q.shape == (M, K) and q.stride(0) % 16 == 0
    a = x.double().abs().amax(dim=1)
    assert torch.equal(s.cpu(), a.float() / 127)
    # 127 x is exact in 64 bits and the quotient, if it is not a half, is 2^-20 away from one
    want = torch.round(x.double() * 127 / a.clamp(min=1e-300)[:, None])
    assert torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_halves_go_to_even(dtype):
    # a = 2 x 127 j / (2 i + 1) makes 127 x / a a half for x = j; and x = a / 2 gives 63.5 for every a
    rows = []
    g = torch.Generator().manual_seed(1)
    for a in [127.0, 254.0, 1.0, 1.5, 0.7, 100.0, 3.2e-5, 6e4] + (torch.rand(24, generator=g) * 50).tolist():
        a = float(torch.tensor(a, dtype=dtype))
        r = torch.cat([torch.tensor([a, a / 2, -a / 2, a / 4, -a * 0.75]), torch.arange(-20, 21) * 0.5 * a / 127,
                       torch.arange(-9, 10) * a / 254])
        rows.append(r.to(dtype))
    x = torch.stack(rows)
    q, _ = sk.int8_quantize(x.to(DEV))
    for i in range(x.shape[0]):
        assert q[i].cpu().tolist() == _codes(x[i]), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_mantissa(dtype):
    """Every mantissa of the row's maximum against every mantissa of x down to 2^-8 of it."""
    n = 1024 if dtype == torch.float16 else 128
    a = torch.arange(n, 2 * n)                                   # row maxima, a / n in [1, 2)
    X, shift = torch.meshgrid(torch.arange(n, 2 * n), torch.arange(0, 9), indexing="ij")
    X, den = X.flatten(), (1 << shift).flatten()                 # x = X / (n den)
    num = torch.where(X[None, :] <= a[:, None] * den[None, :], X[None, :], 0)
    x = torch.cat([a[:, None].double() / n, num.double() / den / n], dim=1).to(dtype)
    x[:, 1::2] *= -1
    q, _ = sk.int8_quantize(x.to(DEV))
    d = (a[:, None] * den[None, :])                              # |Q| = 127 num / d
    f, r = torch.div(127 * num, d, rounding_mode="floor"), (127 * num) % d
    want = f + ((2 * r > d) | ((2 * r == d) & (f % 2 == 1))).long()
    assert torch.equal(q[:, 1:].cpu().long().abs(), want)
    assert bool((q[:, 0] == 127).all()) and not bool((q[:, 1::2] > 0).any())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_extreme_rows(dtype):
    big, tiny = torch.finfo(dtype).max, float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    g = torch.Generator().manual_seed(2)
    x = torch.zeros(8, 48, dtype=dtype)
    x[1] = (torch.rand(48, generator=g) * 2 - 1).to(dtype) * big
    x[1, 0] = big
    x[2] = torch.randint(-9, 10, (48,), generator=g).to(dtype) * tiny        # subnormals only
    x[3, 5] = float("nan")
    x[4, 6] = float("-inf")
    x[5, 7], x[5, 8] = float("nan"), float("inf")
    x[6, 9] = tiny
    x[7, 0], x[7, 1] = -big, tiny
    q, s = sk.int8_quantize(x.to(DEV))
    q, s = q.cpu(), s.cpu()
    for i in (0, 1, 2, 6, 7):
        assert q[i].tolist() == _codes(x[i]), i
        assert s[i] == x[i].double().abs().max().float() / 127
    for i in (3, 4, 5):
        assert bool(s[i].isnan()) and not q[i].any()


def test_quantiser_strides():
    x = torch.randn(70, 400, dtype=torch.float16, device=DEV)
    for v in (x[:, :256], x[:, 3:260], x[::2, 8:264], x.t()[:, :64]):
        q, s = sk.int8_quantize(v)
        q2, s2 = sk.int8_quantize(v.contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)


def test_refusals():
    A, B, sa, sb = (t.to(DEV) for t in _case(32, 64, 128, seed=1))
    for bad, err in (((A.cpu(), B, sa, sb), ValueError), ((A, B.half(), sa, sb), TypeError),
                     ((A, B[:, :64], sa, sb), ValueError), ((A, B, sa[:3], sb), ValueError),
                     ((A, B, sa.half(), sb), TypeError), ((A, B, sa, sb.cpu()), ValueError),
                     ((A[0], B, sa, sb), ValueError), ((A[:0], B, sa[:0], sb), ValueError),
                     ((A[:, :0], B[:, :0], sa, sb), ValueError)):
        with pytest.raises(err):
            sk.streamk_int8_nt(*bad)
    with pytest.raises(TypeError):
        sk.streamk_int8_nt(A, B, sa, sb, out_dtype=torch.float32)
    with pytest.raises(TypeError):
        sk.streamk_int8_nt(A, B, sa, sb, fixup="atomic")
    with pytest.raises(sk.StreamKError):
        sk.streamk_int8_nt(A, B, sa, sb, tile_m=256, tile_n=48)      # CTA pairs: steps of 32
    with pytest.raises(ValueError):
        sk.streamk_int8_nt(A, B, sa, sb, out=torch.empty(32, 65, dtype=torch.float16, device=DEV))
    for bad, err in ((A, TypeError), (torch.zeros(2, 8), ValueError), (torch.zeros(8, dtype=torch.half, device=DEV), ValueError),
                     (torch.zeros(0, 8, dtype=torch.half, device=DEV), ValueError),
                     (torch.zeros(8, 0, dtype=torch.half, device=DEV), ValueError)):
        with pytest.raises(err):
            sk.int8_quantize(bad)


def test_quantised_layer_is_near_the_unquantised_one():
    """Quantiser and product together: each operand's codes are off by at most half a step, i.e.
    scale / 2, so |C - X W^T| <= sum_k (|x| s_w / 2 + |w| s_x / 2 + s_x s_w / 4), plus the result's
    own rounding (2^-11 relative for fp16) and three fp32 roundings."""
    g = torch.Generator().manual_seed(4)
    X, W = torch.randn(50, 1024, generator=g).half(), (torch.randn(300, 1024, generator=g) * 0.02).half()
    qx, sx = sk.int8_quantize(X.to(DEV))
    qw, sw = sk.int8_quantize(W.to(DEV))
    C = sk.streamk_int8_nt(qx, qw, sx, sw).cpu().double()
    ref = X.double() @ W.double().T
    sx, sw = sx.cpu().double()[:, None], sw.cpu().double()[None, :]
    bound = X.double().abs().sum(1)[:, None] * sw / 2 + W.double().abs().sum(1)[None, :] * sx / 2 + 1024 * sx * sw / 4
    assert bool(((C - ref).abs() <= bound * (1 + 1e-6) + C.abs() * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -24).all())
    assert oracle.rel_err(C, ref) <= 2e-2


def test_addresses_beyond_32_bits():
    """More than 2^31 elements in the result, in the weights and in the quantised rows; what lies behind
    them is compared with small calls on copies."""
    g = torch.Generator(device=DEV).manual_seed(2)

    def ints(*shape):
        return torch.randint(-128, 128, shape, generator=g, device=DEV, dtype=torch.int8)

    for M, N, K in ((70_000, 33_000, 80), (20, 33_000, 70_000), (3, 33_000, 70_000), (33_000, 20, 70_000)):
        A, B = ints(M, K), ints(N, K)
        sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV)
        got = sk.streamk_int8_nt(A, B, sa, sb, out_dtype=torch.bfloat16)
        sk.check_status()
        for rows in (slice(0, 3), slice(M - 3, M)):
            for cols in (slice(0, 20), slice(N - 20, N)):
                ref = _ref(*(t.cpu() for t in (A[rows], B[cols], sa[rows], sb[cols])), torch.bfloat16)
                assert torch.equal(_bits(got[rows, cols].contiguous()), _bits(ref)), (M, N, K, rows, cols)
        del A, B, got
    X = torch.empty(530_000, 4104, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    q, s = sk.int8_quantize(X)
    for rows in (slice(0, 5), slice(523_270, 523_275), slice(529_995, 530_000)):
        q1, s1 = sk.int8_quantize(X[rows].clone())
        assert torch.equal(q[rows], q1) and torch.equal(s[rows], s1)
