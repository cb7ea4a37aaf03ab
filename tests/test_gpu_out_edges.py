"""`out` as a part of a wider buffer: nothing beside it is written, whatever column the result ends at.
(TMA stores are clipped to whole 16 bytes, not to the matrix's last column.)"""
import pytest
import torch

import streamk_b200 as sk

pytestmark = pytest.mark.gpu
DEV = "cuda"
MARK = 7.0


def _beside(buf, out):
    """What lies beside `out`, after `out` itself has been marked like the rest."""
    out.fill_(MARK)
    return bool((buf == MARK).all())


@pytest.mark.parametrize("M", [1, 40, 100, 257, 2049])
@pytest.mark.parametrize("N", [37, 65, 77, 70, 250, 251, 259, 1029, 2000])
def test_int8(M, N):
    K = 208
    g = torch.Generator(device=DEV).manual_seed(M + N)
    A, B = (torch.randint(-128, 128, (r, K), generator=g, device=DEV, dtype=torch.int8) for r in (M, N))
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV) * 0.01
    want = (((A.double() @ B.double().T).float() * sa[:, None]) * sb[None, :])
    up8 = -(-N // 8) * 8
    for pitch, first in ((up8, 0), (up8 + 8, 8), (up8 + 64, 0), (N + 1, 0), (N + 3, 3)):
        for dtype in (torch.float16, torch.bfloat16):
            buf = torch.full((M + 1, max(pitch, N + first)), MARK, dtype=dtype, device=DEV)
            out = buf[:M, first:first + N]
            for kw in ({}, {"schedule": "dp"}, {"schedule": "streamk"}, {"schedule": "hybrid"},
                       {"tile_m": 256, "tile_n": 256, "schedule": "dp"}, {"tile_m": 256, "tile_n": 96, "schedule": "dp"},
                       {"tile_m": 128, "tile_n": 64, "schedule": "dp"}, {"tile_m": 128, "tile_n": 80, "schedule": "dp"}):
                sk.streamk_int8_nt(A, B, sa, sb, out=out, out_dtype=dtype, **kw)
                assert torch.equal(out, want.to(dtype)), (pitch, first, dtype, kw)
                assert _beside(buf, out), (pitch, first, dtype, kw)
    sk.check_status()


def test_int8_units_of_two_tiles():
    """The largest schedule: 256 x 512 units, the last of which the matrix ends in."""
    M, N, K = 5000, 3001, 256
    g = torch.Generator(device=DEV).manual_seed(0)
    A, B = (torch.randint(-128, 128, (r, K), generator=g, device=DEV, dtype=torch.int8) for r in (M, N))
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV) * 0.01
    want = (((A.double() @ B.double().T).float() * sa[:, None]) * sb[None, :]).half()
    for pitch in (3008, 3080, 3002):
        buf = torch.full((M, pitch), MARK, dtype=torch.float16, device=DEV)
        for schedule in ("auto", "hybrid", "dp"):
            sk.streamk_int8_nt(A, B, sa, sb, out=buf[:, :N], schedule=schedule)
            assert torch.equal(buf[:, :N], want), (pitch, schedule)
            assert _beside(buf, buf[:, :N]), (pitch, schedule)
    sk.check_status()


@pytest.mark.parametrize("kind", ["nt", "nn", "tn"])
@pytest.mark.parametrize("N", [1, 5, 8, 37, 63, 65, 70, 131, 250, 257, 516])
def test_grouped(kind, N):
    sizes, K = [70, 0, 1, 300], 77
    T, E = sum(sizes), len(sizes)
    g = torch.Generator(device=DEV).manual_seed(N)
    run = {"nt": sk.streamk_grouped_nt, "nn": sk.streamk_grouped_nn, "tn": sk.streamk_grouped_tn}[kind]
    A = torch.randn(T, K, generator=g, device=DEV).half()
    B = torch.randn(*((T, N) if kind == "tn" else (E, N, K) if kind == "nt" else (E, K, N)), generator=g, device=DEV).half()
    off = torch.tensor([sum(sizes[:i]) for i in range(E + 1)], device=DEV)
    for dtype in (torch.float16, torch.float32) if kind == "tn" else (torch.float16,):
        kw = {"out_dtype": dtype} if kind == "tn" else {}
        want = run(A, B, off, **kw)
        unit = 16 // dtype.itemsize
        up = -(-N // unit) * unit
        rows = (E, K + 1) if kind == "tn" else (T + 1,)
        for pitch, first in ((up, 0), (up + unit, unit), (up + 64, 0), (N + 1, 0), (N + 3, 1)):
            buf = torch.full((*rows, max(pitch, N + first)), MARK, dtype=dtype, device=DEV)
            out = buf[..., :-1, first:first + N]
            run(A, B, off, out=out, **kw)
            assert torch.equal(out, want), (dtype, pitch, first)
            assert _beside(buf, out), (dtype, pitch, first)
    sk.check_status()


@pytest.mark.parametrize("schedule", ["auto", "dp", "streamk", "hybrid", "cluster"])
@pytest.mark.parametrize("M,N", [(1, 37), (40, 65), (100, 77), (300, 251), (600, 1029)])
def test_16_bit_products(M, N, schedule):
    K = 512
    g = torch.Generator(device=DEV).manual_seed(M)
    A, B = (torch.randn(r, K, generator=g, device=DEV).half() for r in (M, N))
    up8 = -(-N // 8) * 8
    for pitch, first in ((up8, 0), (up8 + 8, 8), (N + 1, 0)):
        buf = torch.full((M + 1, max(pitch, N + first)), MARK, dtype=torch.float16, device=DEV)
        out = buf[:M, first:first + N]
        try:
            sk.streamk_fp16_nt(A, B, out=out, schedule=schedule)
        except sk.StreamKError as e:                     # (cluster: too many tiles)
            assert schedule == "cluster" and e.status == 3
            continue
        assert float((out.float() - A.float() @ B.float().T).abs().max()) <= 0.2
        assert _beside(buf, out), (pitch, first)
    sk.check_status()
