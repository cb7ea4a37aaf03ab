"""Host side of the 8-bit integer and grouped entry points, without a GPU: refusals of the C ABI and
of the Python layer, the plans that `auto` picks, the shortcut module's fall-through."""
import ctypes as C

import pytest
import torch

import streamk_b200 as sk
from streamk_b200 import _lib as L

FAKE = 1 << 20          # an aligned address that is never read: every call here is refused before a launch


def _i8(lib, A=FAKE, B=FAKE, sa=FAKE, sb=FAKE, out=FAKE, **kw):
    f = dict(M=4, N=16, K=64, lda=64, ldb=64, ldc=16, layout=1, schedule=4, fixup=1)
    f.update(kw)
    return lib.sk_gemm_i8(C.byref(L.SkProblem(**f)), A, B, sa, sb, out, FAKE, 1 << 40, None)


def test_int8_refusals(lib):
    assert lib.sk_gemm_i8(None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == L.SK_ERR_ARG
    for kw in (dict(A=None), dict(B=None), dict(sa=None), dict(sb=None), dict(out=None), dict(layout=0), dict(layout=2),
               dict(fixup=0)):
        assert _i8(lib, **kw) == L.SK_ERR_ARG, kw
    for kw in (dict(M=0), dict(N=0), dict(K=0), dict(K=-5), dict(lda=48), dict(ldb=63)):
        assert _i8(lib, **kw) == L.SK_ERR_SHAPE, kw
    for kw in (dict(lda=72), dict(ldb=65), dict(sa=FAKE + 2), dict(sb=FAKE + 1)):
        assert _i8(lib, **kw) == L.SK_ERR_ALIGN, kw
    for kw in (dict(K=131072, lda=131072, ldb=131072), dict(M=0x7fff0001), dict(N=0x7fffffff, ldc=0x7fffffff)):
        assert _i8(lib, **kw) == L.SK_ERR_LIMIT, kw


def _quant(lib, X=FAKE, M=2, K=8, ldx=8, Q=FAKE, ldq=16, s=FAKE):
    return lib.sk_quantize_i8(X, M, K, ldx, 0, Q, ldq, s, None)


def test_quantiser_refusals(lib):
    for kw in (dict(X=None), dict(Q=None), dict(s=None)):
        assert _quant(lib, **kw) == L.SK_ERR_ARG, kw
    for kw in (dict(M=0), dict(K=0), dict(ldx=7), dict(ldq=7), dict(M=-1)):
        assert _quant(lib, **kw) == L.SK_ERR_SHAPE, kw
    for kw in (dict(X=FAKE + 1), dict(s=FAKE + 2)):
        assert _quant(lib, **kw) == L.SK_ERR_ALIGN, kw


def _grouped(lib, A=FAKE, B=FAKE, off=FAKE, out=FAKE, ws=FAKE, **kw):
    f = dict(kind=0, T=8, E=2, N=16, K=32, lda=32, ldb=32, ldc=16, stride_b=512, stride_c=512)
    f.update(kw)
    return lib.sk_gemm_grouped(C.byref(L.SkGroupedProblem(**f)), A, B, off, out, ws, 1 << 40, None)


def test_grouped_refusals(lib):
    assert lib.sk_gemm_grouped(None, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == L.SK_ERR_ARG
    for kw in (dict(A=None), dict(B=None), dict(off=None), dict(out=None), dict(kind=3), dict(kind=-1),
               dict(flags=L.SK_FLAG_OUT_F32)):
        assert _grouped(lib, **kw) == L.SK_ERR_ARG, kw
    for kw in (dict(T=0), dict(E=0), dict(N=0), dict(K=0), dict(lda=24), dict(ldb=24), dict(ldc=15), dict(stride_b=511),
               dict(ldb=33),   # (16 rows of 33 do not fit the 512 between two groups)
               dict(kind=1, ldb=8), dict(kind=2, ldb=8), dict(kind=2, stride_c=511)):
        assert _grouped(lib, **kw) == L.SK_ERR_SHAPE, kw
    wide = dict(ldb=0x7ffffff8, ldc=0x7fffffff, stride_b=1 << 40, stride_c=1 << 40)
    for kw in (dict(E=1025), dict(T=0x7fff0001), dict(N=0x7fff0001, stride_b=1 << 40, ldc=0x7fffffff),
               dict(kind=1, N=0x7fffffff, **wide), dict(kind=2, N=0x7fffffff, **wide),
               dict(kind=2, K=0x7fff0001, lda=1 << 31, stride_c=1 << 40)):
        assert _grouped(lib, **kw) == L.SK_ERR_LIMIT, kw
    for kw in (dict(A=FAKE + 8), dict(B=FAKE + 2), dict(lda=36), dict(ldb=33, stride_b=528), dict(stride_b=516), dict(out=FAKE + 1),
               dict(off=FAKE + 2), dict(off=FAKE + 4, flags=L.SK_FLAG_OFFSETS_64),
               dict(kind=2, out=FAKE + 2, flags=L.SK_FLAG_OUT_F32)):
        assert _grouped(lib, **kw) == L.SK_ERR_ALIGN, kw


def test_cpu_tensors_are_refused():
    h, q = torch.zeros(4, 32, dtype=torch.half), torch.zeros(4, 32, dtype=torch.int8)
    s, off = torch.ones(4), torch.tensor([0, 4])
    for call in (lambda: sk.int8_quantize(h), lambda: sk.streamk_int8_nt(q, q, s, s),
                 lambda: sk.streamk_grouped_nt(h, h[None], off), lambda: sk.streamk_grouped_nn(h, h[None], off),
                 lambda: sk.streamk_grouped_tn(h, h, off)):
        with pytest.raises(ValueError):
            call()


def test_the_shortcut_hands_back_what_it_does_not_take():
    m = L.load_host()
    h = torch.zeros(4, 32, dtype=torch.half)
    for args in ((), (None,), (h,), (h.numpy(),), (h, h)):
        assert m.quantize(*args) is None
    for args in ((), (h, h, h, h, True), (None,) * 5, (3, "x", 1, 2, False)):
        assert m.gemm_i8(*args) is None
    for args in ((), (0, h, h, h, False), (2, None, None, None, True)):
        assert m.grouped(*args) is None
    with pytest.raises(TypeError):
        m.set_workspace(1)
    with pytest.raises(TypeError):
        m.grouped("nt", h, h, h, False)


def test_workspace_header(lib):
    assert lib.sk_workspace_header_bytes(0) == 0
    assert 256 + 16 * 148 <= lib.sk_workspace_header_bytes(148) < 1 << 16
    assert lib.sk_stream_capture_id(None, None) == L.SK_ERR_ARG


@pytest.mark.parametrize("shape,name,tile", [
    ((1, 11008, 4096), "gemv", None), ((16, 4096, 11008), "cluster", (16, 128)), ((16, 11008, 4096), "gemv", None), ((8, 4096, 11008), "gemv", None), ((16, 28672, 8192), "dp", None),
    ((24, 4096, 4096), "cluster", None), ((48, 512, 512), "dp", (128, 64)), ((44, 2176, 2208), "cluster", (48, 128)),
    ((100, 512, 8192), "cluster", (128, 64)), ((100, 2048, 8192), "cluster", (128, 64)), ((100, 2048, 4096), "dp", (128, 64)), ((48, 28672, 1024), "dp", (128, 256)),
    ((100, 4096, 4096), "dp", (128, 64)), ((400, 4096, 4096), "dp", (128, 128)), ((128, 28672, 1024), "dp", (128, 256)),
    ((200, 12288, 4096), "dp", (256, 192)), ((800, 12288, 4096), "dp", (256, 256)), ((8192, 28672, 8192), "dp", (256, 256))])
def test_auto_plans(shape, name, tile):
    p = sk.schedule_info(*shape, kind="int8")
    assert sk.SCHEDULE_NAMES[p["schedule"]] == name
    if tile:
        assert (p["tile_m"], p["tile_n"]) == tile


def test_no_more_clusters_than_are_resident():
    for N, size in ((14 * 64, 8), (15 * 64, 4), (32 * 64, 4), (33 * 64, 2)):
        assert sk.schedule_info(100, N, 8192, kind="int8", schedule="cluster", tile_m=128, tile_n=64)["cluster"] == size


def test_every_tile_is_walked_once_under_every_schedule():
    """The plans that sk_gemm_i8 makes cover K and the tiles: units of 128 of K, odd sizes included."""
    for shape in ((3, 77, 129), (300, 1000, 1000), (1000, 4104, 257)):
        for schedule in ("streamk", "hybrid", "dp"):
            p = sk.schedule_info(*shape, kind="int8", schedule=schedule)
            assert p["tile_k"] == 128 and p["iters_per_tile"] == -(-shape[2] // 128)
            assert p["tiles_m"] * p["tile_m"] >= shape[0] and p["tiles_n"] * p["tile_n"] >= shape[1]
    with pytest.raises(sk.StreamKError):
        sk.schedule_info(1, 16, 131072, kind="int8")
