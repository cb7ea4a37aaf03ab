"""Python operator surface: the reference's entry points, backed by the C ABI.

The reference (LeiWang1999/Stream-k.tvm) has no importable API; each script
builds `tl_matmul_streamk(...)` and calls `tl_mod(A, B, C)` on CUDA tensors
(streamk_fp32.py:57-202, streamk_fp16.py:116-387, streamk_fp16_ladder.py,
streamk_fp16_ladder_block_reduce_q4.py).  The functions here keep those names
and argument meanings (A [M,K]; B [K,N] for NN, [N,K] for NT; C [M,N]) but
return a fresh C instead of accumulating into a pre-zeroed one.

Everything runs on the GPU through libstreamk_b200.so; there is no CPU path.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import warnings
from dataclasses import dataclass

import torch

from . import _lib as L

__all__ = [
    "streamk_fp32", "streamk_fp16_nn", "streamk_fp16_nt", "streamk_fp16_nt_host", "streamk_fp16_atomic",
    "streamk_fp16_block_reduce", "ladder_prepack", "streamk_fp16_ladder",
    "streamk_fp16_ladder_block_reduce", "q4_prepack", "dequant_w4",
    "streamk_fp16_ladder_block_reduce_q4", "int8_quantize", "streamk_int8_nt",
    "streamk_grouped_nt", "streamk_grouped_nn", "streamk_grouped_tn", "schedule_info", "check_status",
    "SCHEDULE_NAMES", "reset_workspace", "release_cached_memory", "cached_memory_bytes", "device_info", "LadderWeight", "PackedQ4", "StreamKError", "SCHEDULES", "FIXUPS",
]

StreamKError = L.StreamKError
SCHEDULES = L.SCHEDULES   # name -> SK_SCHED_* value
FIXUPS = L.FIXUPS
SCHEDULE_NAMES = {v: k for k, v in L.SCHEDULES.items()}   # SK_SCHED_* value -> name
GROUP_SIZE = 128


# --------------------------------------------------------------------------- state
class _Workspace:
    __slots__ = ("buf", "nbytes", "ptr", "status_host")

    def __init__(self, device: torch.device, stream_ptr: int):
        lib = L.load()
        sms = torch.cuda.get_device_properties(device).multi_processor_count
        self.nbytes = int(lib.sk_workspace_bytes(sms))
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        self.ptr = self.buf.data_ptr()
        self.status_host = torch.zeros(8, dtype=torch.int32).pin_memory()   # this workspace's, the device's
        L.check(lib.sk_workspace_init(self.buf.data_ptr(), self.nbytes, stream_ptr),
                "sk_workspace_init")


# Device memory this module keeps between calls: one workspace (sk_workspace_bytes, about
# 57 MB on 148 SMs) per (device, stream) that ever launched a GEMM, and the staging buffers of
# streamk_fp16_nt_host per (device, shape, slab).  cached_memory_bytes() reports them,
# release_cached_memory() drops them.
_workspaces: dict[tuple[int, int], _Workspace] = {}


# The host side of a call costs more than many of the kernels: the raw stream handle comes
# straight from the runtime binding where torch has it (0.1 us against 2.4), and the device is
# switched only if another one is current (1.5 us a switch).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(device: torch.device) -> int:
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device() if device.index is None else device.index)
    return int(torch.cuda.current_stream(device).cuda_stream)


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """Context manager: `device` is current inside."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


# The fast path from tensors to the C ABI (csrc/host/sk_torch_host.cpp): int8_quantize,
# streamk_int8_nt and the grouped products offer it their arguments first; it returns None where
# there is anything to check, copy or refuse, and the code below takes over.  Where it cannot be
# built or loaded the code below does it all, at 11-14 us of host time a call instead of 4-5.
_fast = None


class _NoShortcut:
    """Stands in for the module: takes nothing."""
    @staticmethod
    def _none(*args):
        return None
    quantize = gemm_i8 = grouped = set_workspace = clear_workspaces = set_captured = _none


def _load_fast():
    global _fast
    L.load()                 # (the kernels themselves: an error if they are missing)
    try:
        _fast = L.load_host()
    except (ImportError, OSError, RuntimeError) as e:
        warnings.warn(f"calls take the longer host path: the host module could not be loaded ({e})", RuntimeWarning,
                      stacklevel=3)
        _fast = _NoShortcut()
    _fast.clear_workspaces()
    for (device, stream), ws in _workspaces.items():
        _fast.set_workspace(device, stream, ws.ptr, ws.nbytes)
    for device in _capture_ws:
        _fast.set_captured(device, True)
    return _fast


def _workspace(device: torch.device) -> _Workspace:
    """One workspace per (device, stream): launches that may overlap never share one."""
    key = (device.index if device.index is not None else torch.cuda.current_device(),
           _stream_ptr(device))
    ws = _workspaces.get(key)
    if ws is None:
        with torch.cuda.device(device):
            ws = _Workspace(device, key[1])
        ws = _workspaces.setdefault(key, ws)   # (another thread may have been first: one for both, and the shortcut's)
        if _fast is not None:
            _fast.set_workspace(key[0], key[1], ws.ptr, ws.nbytes)
    return ws


# Captured calls of the 8-bit integer and grouped products do not use the stream's workspace: graphs
# are often captured on one stream and replayed on several at a time, and would share it.  Each
# capture gets workspaces of its own, one for each stream that it records (its branches may run at
# the same time), allocated while capturing and therefore in the graph's memory pool, whose
# counters a node of the graph zeroes at the start of every replay.  They are held until another
# capture begins or one of these products is called outside one; from then on they belong to the
# graph like any tensor that its capture made and let go.  Errors of a replay are therefore not reported in them
# but in the device's own status word (SK_FLAG_DEVICE_STATUS), which check_status() reads too.
_capture_ws: dict[int, tuple[int, dict[int, torch.Tensor]]] = {}     # device -> capture id, stream -> workspace


def _call_workspace(device: torch.device) -> tuple[int, int, int]:
    """Workspace of a call that may be captured: its address, its size, the flags that go with it."""
    stream = _stream_ptr(device)
    lib = L.load()
    cid = C.c_ulonglong(0)
    L.check(lib.sk_stream_capture_id(stream, C.byref(cid)), "sk_stream_capture_id")
    if cid.value == 0:
        if _capture_ws.pop(device.index, None) is not None and _fast is not None:
            _fast.set_captured(device.index, False)
        ws = _workspace(device)
        return ws.ptr, ws.nbytes, 0
    held = _capture_ws.get(device.index)
    if held is None or held[0] != cid.value:
        held = _capture_ws[device.index] = (cid.value, {})
        if _fast is not None:   # (the next eager call on this device comes here, too)
            _fast.set_captured(device.index, True)
    buf = held[1].get(stream)
    if buf is None:
        sms = torch.cuda.get_device_properties(device).multi_processor_count
        buf = torch.empty(int(lib.sk_workspace_bytes(sms)), dtype=torch.uint8, device=device)
        L.check(lib.sk_workspace_init(buf.data_ptr(), int(lib.sk_workspace_header_bytes(sms)), stream), "sk_workspace_init")
        held[1][stream] = buf
    return buf.data_ptr(), buf.numel(), L.SK_FLAG_DEVICE_STATUS


def reset_workspace(device=None) -> None:
    """Re-zero the workspace of the current stream (needed after a device-reported error)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    ws = _workspace(device)
    with torch.cuda.device(device):
        L.check(L.load().sk_workspace_init(ws.buf.data_ptr(), ws.nbytes, _stream_ptr(device)),
                "sk_workspace_init")


def cached_memory_bytes() -> int:
    """Device bytes held by the cached workspaces and host-pipeline staging buffers."""
    n = sum(ws.nbytes for ws in _workspaces.values())
    n += sum(buf.numel() for _, held in _capture_ws.values() for buf in held.values())
    for pipe in _host_pipes.values():
        n += pipe.nbytes
    return n


def release_cached_memory() -> None:
    """Drop every cached workspace and staging buffer (all devices).  Synchronises the devices
    first, so nothing in flight still uses them; the next call allocates afresh."""
    for dev in {k[0] for k in _workspaces} | {k[0] for k in _host_pipes}:
        torch.cuda.synchronize(dev)
    if _fast is not None:
        _fast.clear_workspaces()
    _workspaces.clear()
    _capture_ws.clear()
    _host_pipes.clear()


def check_status(device=None) -> None:
    """Synchronise the current stream and raise if a kernel reported an error: one of this stream's,
    or one of a call of the 8-bit integer or grouped products that was captured into a graph (whatever
    stream replayed it; the replays of other streams may not have finished)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    ws = _workspace(device)
    lib = L.load()
    with torch.cuda.device(device):
        captured = C.c_void_p()
        L.check(lib.sk_device_status(C.byref(captured)), "sk_device_status")
        for i, status in enumerate((ws.ptr, captured)):
            st = C.cast(ws.status_host.data_ptr() + 16 * i, C.POINTER(L.SkStatus))
            L.check(lib.sk_poll_status(status, st, _stream_ptr(device)), "sk_poll_status")
        torch.cuda.current_stream(device).synchronize()
    words = [int(x) & 0xFFFFFFFF for x in ws.status_host.tolist()]
    where, (code, cta, d0, d1) = "device status", words[:4]
    if code != L.SK_OK:
        reset_workspace(device)
    elif words[4] != L.SK_OK:     # (with both, this one is left for the next check)
        where, (code, cta, d0, d1) = "device status of a captured call", words[4:]
        with torch.cuda.device(device):
            L.check(lib.sk_workspace_init(captured, L.SK_DEVICE_STATUS_BYTES, _stream_ptr(device)), "sk_workspace_init")
    if code != L.SK_OK:
        raise StreamKError(code, where, f"[cta {cta}, detail {d0}, {d1}]")


def device_info(device: int = 0) -> dict:
    info = L.SkDeviceInfo()
    st = L.load().sk_query(device, C.byref(info))
    d = {n: getattr(info, n) for n, _ in info._fields_}
    d["status"] = st
    return d


# --------------------------------------------------------------------------- helpers
_OPTION_KEYS = ("tile_m", "tile_n", "num_sms", "group_m", "out", "timeout_us", "pdl", "no_table",
                "_drop_flag_cta", "_bf16")


_NO_OPTIONS = dict.fromkeys(_OPTION_KEYS)


def _options(kw: dict) -> dict:
    """Common keyword arguments of every GEMM entry point:
    tile_m / tile_n  tile extents (None = choose; tile_m < 128 puts the weights on the UMMA
                     M dimension, the short-M form), num_sms (grid bound), group_m (tile
                     rasterisation), out (result buffer, which shares no element with the operands),
                     timeout_us (bound of every device
                     wait), pdl (True: programmatic dependent launch, the kernel's start-up may
                     overlap the tail of the previous kernel of the stream; fp16 / W4A16),
                     no_table (True: schedule "auto" by the built-in rules only, ignoring the table
                     of tuned shapes),
                     _drop_flag_cta (test hook: index of a CTA that withholds its flag)."""
    if not kw:
        return _NO_OPTIONS.copy()
    unknown = set(kw) - set(_OPTION_KEYS)
    if unknown:
        raise TypeError(f"unexpected keyword argument(s): {sorted(unknown)}")
    return {k: kw.get(k) for k in _OPTION_KEYS}


def _problem(M, N, K, lda, ldb, ldc, layout, schedule, fixup, o: dict) -> L.SkProblem:
    if schedule not in L.SCHEDULES:
        raise ValueError(f"schedule must be one of {sorted(L.SCHEDULES)}, got {schedule!r}")
    if fixup not in L.FIXUPS:
        raise ValueError(f"fixup must be one of {sorted(L.FIXUPS)}, got {fixup!r}")
    if (M | N | K | lda | ldb | ldc) > 0x7fffffff:   # (ctypes would take them modulo 2^32)
        _check_int32(M=M, N=N, K=K, pitch_a=lda, pitch_b=ldb, pitch_out=ldc)
    # (positional: the fields of sk_problem in order; half the time of keywords)
    return L.SkProblem(M, N, K, lda, ldb, ldc, L.LAYOUTS[layout], L.SCHEDULES[schedule], L.FIXUPS[fixup],
                       int(o["tile_m"] or 0), int(o["tile_n"] or 0), int(o["num_sms"] or 0), int(o["group_m"] or 0),
                       int(o["timeout_us"] or 0),
                       # (the C field is 0 = off, n = CTA n - 1)
                       0 if o["_drop_flag_cta"] is None else int(o["_drop_flag_cta"]) + 1,
                       (L.SK_FLAG_PDL if o["pdl"] else 0) | (L.SK_FLAG_NO_TABLE if o["no_table"] else 0)
                       | (L.SK_FLAG_BF16 if o["_bf16"] else 0))


def schedule_info(M: int, N: int, K: int, *, kind: str = "f16", schedule: str = "auto",
                  num_sms: int = 148, gather_peers: int = 0, **kw) -> dict:
    """Host scheduler integers (streamk_fp16.py:83-113) and the tile plan for a problem;
    needs no GPU.  kind: "f32", "f16" (what the fp16 NT entry point runs: single-CTA tiles, or
    for large problems the CTA-pair kernel, described over num_sms / 2 pairs), "w4a16", or
    "f16_pairs" (the CTA-pair kernel with num_sms pairs), or "int8" (what the 8-bit integer
    entry point runs).  gather_peers > 0: the plan of the
    fused all-gather call with that many peers."""
    o = _options(kw)
    prob = _problem(M, N, K, K, K, N, "nt", schedule, "atomic", o)
    info = L.SkScheduleInfo()
    kinds = {"f32": 0, "f16": 1, "w4a16": 2, "f16_pairs": 3, "int8": 4}
    if gather_peers:
        L.check(L.load().sk_schedule_gather(C.byref(prob), gather_peers, num_sms, C.byref(info)),
                "sk_schedule_gather")
    else:
        L.check(L.load().sk_schedule(C.byref(prob), kinds[kind], num_sms, C.byref(info)), "sk_schedule")
    return info.as_dict()


HALF_TYPES = (torch.float16, torch.bfloat16)


def _check_matrix(name: str, t: torch.Tensor, dtype) -> None:
    """dtype: one torch dtype, or a tuple of acceptable ones."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this library has no CPU path)")
    ok = t.dtype in dtype if isinstance(dtype, tuple) else t.dtype == dtype
    if not ok:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")


def _rowmajor(t: torch.Tensor) -> torch.Tensor:
    # The reference asserts contiguity (triton_impl.py:199-201); row-major views
    # with a padded leading dimension are accepted here as well.
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t
    return t.contiguous()


def _out(out, M, N, dtype, device):
    if out is None:   # (empty_strided: 1.7 us on the host, empty 2.4)
        return torch.empty_strided((M, N), (N, 1), dtype=dtype, device=device)
    if out.shape != (M, N) or out.dtype != dtype or out.device != device or out.stride(1) != 1:
        raise ValueError("out must be a row-major [M,N] tensor of the result dtype on A's device")
    return out


def _pad_k8(t: torch.Tensor, k_dim: int) -> torch.Tensor:
    """TMA needs 16-byte row pitches: pad the K extent of an fp16 operand to a multiple of 8."""
    k = t.shape[k_dim]
    pad = (-k) % 8
    if pad == 0:
        return t
    spec = (0, pad) if k_dim == 1 else (0, 0, 0, pad)
    return torch.nn.functional.pad(t, spec)


def _aligned16(t: torch.Tensor) -> torch.Tensor:
    if t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0:
        return t
    n = torch.empty((t.shape[0], (t.shape[1] + 7) // 8 * 8), dtype=t.dtype, device=t.device)
    n[:, : t.shape[1]].copy_(t)
    return n[:, : t.shape[1]]


# --------------------------------------------------------------------------- fp32
def streamk_fp32(A: torch.Tensor, B: torch.Tensor, *, fixup: str = "atomic",
                 schedule: str = "auto", trans_b: bool = False, **kw) -> torch.Tensor:
    """C = A @ B in fp32 (FFMA, no TF32).  A [M,K]; B [K,N] (or [N,K] with trans_b).

    Mirrors `tl_matmul_streamk(..., "float32", "float32", "float32", ...)` of
    streamk_fp32.py:57-202.  `schedule="hybrid"` is the reference's split.
    """
    o = _options(kw)
    _check_matrix("A", A, torch.float32)
    _check_matrix("B", B, torch.float32)
    A = _rowmajor(A)
    B = _rowmajor(B)
    M, K = A.shape
    if trans_b:
        N, Kb = B.shape
    else:
        Kb, N = B.shape
    if K != Kb:
        raise ValueError(f"Incompatible dimensions: A {tuple(A.shape)} B {tuple(B.shape)}")
    Cout = _out(o["out"], M, N, torch.float32, A.device)
    prob = _problem(M, N, K, A.stride(0), B.stride(0), Cout.stride(0), "nt" if trans_b else "nn",
                    schedule, fixup, o)
    with _on(A.device):
        ws = _workspace(A.device)
        L.check(L.load().sk_gemm_f32(C.byref(prob), A.data_ptr(), B.data_ptr(), Cout.data_ptr(),
                                     ws.buf.data_ptr(), ws.nbytes, _stream_ptr(A.device)),
                "sk_gemm_f32")
    return Cout


# --------------------------------------------------------------------------- fp16
def _gemm_f16(A, B, layout, fixup, schedule, kw):
    """fp16 operands, or bfloat16 ones (both operands alike; the result has their type)."""
    o = _options(kw)
    _check_matrix("A", A, HALF_TYPES)
    dtype = A.dtype
    o["_bf16"] = dtype == torch.bfloat16
    M, K = A.shape
    if layout == "ladder":
        if not isinstance(B, LadderWeight):
            raise TypeError("B must come from ladder_prepack()")
        if B.K != K:
            raise ValueError(f"Incompatible dimensions: A {tuple(A.shape)} weight K={B.K}")
        if B.dtype != dtype:
            raise TypeError(f"A is {dtype} but the weight image was packed from {B.dtype}")
        N = B.N
        Bt, ldb = B.data, 0
        A = _aligned16(_rowmajor(_pad_k8(A, 1)))
    else:
        _check_matrix("B", B, dtype)
        if layout == "nt":
            N, Kb = B.shape
        else:
            Kb, N = B.shape
        if K != Kb:
            raise ValueError(f"Incompatible dimensions: A {tuple(A.shape)} B {tuple(B.shape)}")
        A = _aligned16(_rowmajor(_pad_k8(A, 1)))
        if layout == "nt":
            Bt = _aligned16(_rowmajor(_pad_k8(B, 1)))
        else:
            # NN: rows of B are K; the N pitch must be a multiple of 8 halves
            Bt = _aligned16(_rowmajor(_pad_k8(B, 0)))
        ldb = Bt.stride(0)
    Cout = _out(o["out"], M, N, dtype, A.device)
    prob = _problem(M, N, A.shape[1], A.stride(0), ldb, Cout.stride(0), layout, schedule, fixup, o)
    with _on(A.device):
        ws = _workspace(A.device)
        L.check(L.load().sk_gemm_f16(C.byref(prob), A.data_ptr(), Bt.data_ptr(), Cout.data_ptr(),
                                     ws.buf.data_ptr(), ws.nbytes, _stream_ptr(A.device)),
                "sk_gemm_f16")
    return Cout


def streamk_fp16_nt(A, B, *, fixup="block_reduce", schedule="auto", **kw):
    """C = A @ B.T, fp16 in, fp32 accumulate, fp16 out.  A [M,K], B [N,K].
    (bfloat16 tensors are accepted as well, here and in the NN and ladder forms: same kernels,
    bf16 operands, fp32 accumulation, bf16 result; the reference is fp16 only.)

    Mirrors `tl_matmul_streamk(M, N, K, streamk_tiles, "float16", "float16", ...)` +
    `tl_mod(A, B, C)` of streamk_fp16.py:116-387 and streamk_fp16_nt.py:57-192.
    schedule: "auto" (the library picks by shape), "hybrid" (the reference's split),
    "hybrid_dp_first", "streamk", "dp".  fixup: "block_reduce" (deterministic) or "atomic".
    Keyword options: see _options().
    """
    return _gemm_f16(A, B, "nt", fixup, schedule, kw)


class _HostPipe:
    """Device staging buffers, streams and events of streamk_fp16_nt_host for one shape."""

    def __init__(self, M, N, K, slab, device):
        self.key = (M, N, K, slab)
        self.A = torch.empty(M, K, dtype=torch.float16, device=device)
        self.B = [torch.empty(slab, K, dtype=torch.float16, device=device) for _ in range(2)]
        self.C = [torch.empty(M, slab, dtype=torch.float16, device=device) for _ in range(2)]
        self.s_in, self.s_mm, self.s_out = (torch.cuda.Stream(device) for _ in range(3))
        self.nbytes = 2 * (M * K + 2 * slab * K + 2 * M * slab)
        self.busy = None     # event recorded at the end of the last call that used these buffers


_host_pipes: dict[tuple, _HostPipe] = {}
_HOST_PIPES_MAX = 4     # staging sets kept; the least recently used one is dropped beyond that


def streamk_fp16_nt_host(A_host, B_host, out_host=None, *, slabs: int = 8, device=None,
                         fixup="block_reduce", schedule="auto", group=None, **kw):
    """C = A @ B.T for operands and result in (pinned) HOST memory: A [M,K], B [N,K] fp16 CPU
    tensors, result [M,N] fp16 CPU tensor (out_host, or a new pinned tensor).

    Column-sharded use (one process per GPU, `group` = a torch.distributed NCCL group of G
    ranks, B_host / out_host = this rank's column block): A_host is then only this rank's
    1/G of A's rows, [M/G, K]; every rank copies its part from the host and the parts are
    all-gathered into each GPU's memory over NVLink (NCCL, ahead of the first slab's GEMM), so
    that A crosses PCIe once for the whole group instead of once per GPU.

    B and C move in `slabs` column slabs through double-buffered device staging: the
    host-to-device copy of slab i+1, the GEMM of slab i and the device-to-host copy of slab i-1
    run on three streams at once, so a step costs about the larger of the two PCIe directions
    instead of their sum plus the GEMM.  The calling stream waits for the result; the host has
    to synchronise that stream (or the device) before reading out_host.  Each slab is one call of
    streamk_fp16_nt (same keyword options)."""
    for name, t in (("A_host", A_host), ("B_host", B_host)):
        if not isinstance(t, torch.Tensor) or t.is_cuda or t.dtype != torch.float16 or t.dim() != 2:
            raise TypeError(f"{name} must be a 2-D fp16 CPU tensor")
    Mpart, K = A_host.shape
    world = 1
    if group is not None:
        import torch.distributed as dist
        world = dist.get_world_size(group)
    M = Mpart * world
    N = B_host.shape[0]
    if B_host.shape[1] != K:
        raise ValueError("A_host [M,K] and B_host [N,K] disagree on K")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    slabs = max(1, min(int(slabs), N))
    slab = -(-N // slabs)
    slab = (slab + 15) // 16 * 16          # whole 16-column groups: aligned rows in the staging tiles
    slabs = -(-N // slab)
    if out_host is None:
        out_host = torch.empty(M, N, dtype=torch.float16).pin_memory()
    if out_host.shape != (M, N) or out_host.dtype != torch.float16 or out_host.is_cuda or out_host.stride(1) != 1:
        raise ValueError("out_host must be a row-major fp16 CPU tensor of shape [M, N]")
    if not (A_host.is_contiguous() and B_host.is_contiguous()):
        raise ValueError("A_host and B_host must be contiguous")
    key = (device.index, M, N, K, slab)
    pipe = _host_pipes.pop(key, None)
    if pipe is None:
        while len(_host_pipes) >= _HOST_PIPES_MAX:
            old = _host_pipes.pop(next(iter(_host_pipes)))
            if old.busy is not None:
                old.busy.synchronize()      # its last call may still be running
        pipe = _HostPipe(M, N, K, slab, device)
    _host_pipes[key] = pipe                 # (most recently used last)
    cur = torch.cuda.current_stream(device)
    for st in (pipe.s_in, pipe.s_mm, pipe.s_out):
        st.wait_stream(cur)
        # The staging buffers are free again only when the previous call that used them has
        # finished, whichever stream that call was made from.
        if pipe.busy is not None:
            st.wait_event(pipe.busy)
    with torch.cuda.stream(pipe.s_in):
        if world == 1:
            pipe.A.copy_(A_host, non_blocking=True)
        else:
            rank = dist.get_rank(group)
            pipe.A[rank * Mpart:(rank + 1) * Mpart].copy_(A_host, non_blocking=True)
            # row blocks are contiguous: the gather lands in place (NCCL kernel on the copy-in
            # stream; no peer pointer is handed to a GEMM kernel as an operand)
            dist.all_gather_into_tensor(pipe.A, pipe.A[rank * Mpart:(rank + 1) * Mpart], group=group)
    mm_done = [None, None]                  # per staging buffer: GEMM that last read B / wrote C
    out_done = [None, None]                 # per staging buffer: copy-out that last read C
    for i in range(slabs):
        b = i & 1
        n0, n1 = i * slab, min(N, (i + 1) * slab)
        w = n1 - n0
        with torch.cuda.stream(pipe.s_in):
            if mm_done[b] is not None:
                pipe.s_in.wait_event(mm_done[b])
            pipe.B[b][:w].copy_(B_host[n0:n1], non_blocking=True)
            loaded = torch.cuda.Event()
            loaded.record(pipe.s_in)
        with torch.cuda.stream(pipe.s_mm):
            pipe.s_mm.wait_event(loaded)
            if out_done[b] is not None:
                pipe.s_mm.wait_event(out_done[b])
            Cb = pipe.C[b] if w == slab else pipe.C[b][:, :w]
            _gemm_f16(pipe.A, pipe.B[b][:w], "nt", fixup, schedule, dict(kw, out=Cb))
            mm_done[b] = torch.cuda.Event()
            mm_done[b].record(pipe.s_mm)
        with torch.cuda.stream(pipe.s_out):
            pipe.s_out.wait_event(mm_done[b])
            # a pitched DMA straight into the column slab of the row-major host matrix (a strided
            # Tensor.copy_ would go through a staging buffer and a CPU-side scatter)
            L.check(L.load().sk_memcpy2d_async(
                out_host.data_ptr() + n0 * 2, out_host.stride(0) * 2, Cb.data_ptr(), Cb.stride(0) * 2,
                w * 2, M, int(pipe.s_out.cuda_stream)), "sk_memcpy2d_async")
            out_done[b] = torch.cuda.Event()
            out_done[b].record(pipe.s_out)
    cur.wait_stream(pipe.s_out)
    cur.wait_stream(pipe.s_mm)
    cur.wait_stream(pipe.s_in)
    pipe.busy = torch.cuda.Event()
    pipe.busy.record(cur)
    return out_host


def streamk_fp16_nn(A, B, *, fixup="block_reduce", schedule="auto", **kw):
    """C = A @ B, fp16.  A [M,K], B [K,N]  (streamk_fp16_nn.py:57-177)."""
    return _gemm_f16(A, B, "nn", fixup, schedule, kw)


def streamk_fp16_atomic(A, B, **kw):
    """NT GEMM with the order-nondeterministic fp32 red.global.add fixup
    (the role of T.atomic_addx2 in streamk_fp16.py:248-255)."""
    return streamk_fp16_nt(A, B, fixup="atomic", **kw)


def streamk_fp16_block_reduce(A, B, **kw):
    """NT GEMM with the deterministic flag-synchronised fixup.  Keeps the entry name of
    streamk_fp16_block_reduce.py; the intra-CTA split-K it performs there is subsumed by
    TMEM accumulation, the name now denotes the bitwise-reproducible cross-CTA reduction."""
    return streamk_fp16_nt(A, B, fixup="block_reduce", **kw)


@dataclass
class LadderWeight:
    """Weight pre-laid-out by ladder_prepack (opaque image + logical shape)."""
    data: torch.Tensor
    N: int
    K: int
    dtype: torch.dtype = torch.float16


def ladder_prepack(B: torch.Tensor) -> LadderWeight:
    """Re-lay B [N,K] fp16 into the streaming image of the ladder mainloop.

    Replaces `bitblas.ops.LadderPermutate(...)(B.cpu())` (streamk_fp16_ladder.py:468-477);
    runs on the GPU."""
    _check_matrix("B", B, HALF_TYPES)
    B = _rowmajor(B)
    N, K = B.shape
    _check_int32(N=N, K=K, pitch=B.stride(0))
    lib = L.load()
    nbytes = int(lib.sk_ladder_bytes(N, K))
    out = torch.empty(nbytes, dtype=torch.uint8, device=B.device)
    with torch.cuda.device(B.device):
        L.check(lib.sk_prepack_ladder(B.data_ptr(), N, K, B.stride(0), out.data_ptr(), nbytes,
                                      _stream_ptr(B.device)), "sk_prepack_ladder")
    return LadderWeight(out, N, K, B.dtype)


def streamk_fp16_ladder(A, LB: LadderWeight, *, fixup="block_reduce", schedule="auto", **kw):
    """C = A @ W.T with W pre-laid-out (streamk_fp16_ladder.py:137-486)."""
    return _gemm_f16(A, LB, "ladder", fixup, schedule, kw)


def streamk_fp16_ladder_block_reduce(A, LB: LadderWeight, **kw):
    """Ladder path with the deterministic fixup (streamk_fp16_ladder_block_reduce.py)."""
    return streamk_fp16_ladder(A, LB, fixup="block_reduce", **kw)


# --------------------------------------------------------------------------- W4A16
@dataclass
class PackedQ4:
    """uint4 weight + group scales/zeros packed by q4_prepack (opaque image + shape)."""
    data: torch.Tensor
    N: int
    K: int
    group_size: int = GROUP_SIZE     # 32, 64, 128, or 0 = one group per weight row (per-channel)
    signed: bool = False


def q4_prepack(qweight: torch.Tensor, scales: torch.Tensor | None = None,
               zeros: torch.Tensor | None = None, group_size: int = GROUP_SIZE,
               signed: bool = False) -> PackedQ4:
    """Pack 4-bit weights for the W4A16 mainloop.

    qweight: int32 [N, K/8] (nibble j of word w = element 8w+j) or int8/uint8 [N, K/2]
    (low nibble = even k, the reference's storage, …_q4.py:28-30,545-554).
    scales: fp16 [N, K/group_size] or None (=1).  zeros: uint8 [N, K/group_size] in 0..15 or None
    (=0).  With scales=None, zeros=None the GEMM reproduces the reference's `A @ unpack(qB).T`.
    group_size: 128 (the benchmark's), 64, 32, or 0 / K for per-channel scales ([N, 1]).
    signed: the nibbles are two's-complement int4 (-8..7), W = q * s (no zero-points).
    Replaces LadderPermutate + LOP3Permutate on the CPU (…_q4.py:568-595); formats beyond plain
    uint4 have no counterpart in the reference.
    """
    if not qweight.is_cuda:
        raise ValueError("qweight must be a CUDA tensor (this library has no CPU path)")
    if qweight.dtype in (torch.int8, torch.uint8):
        N, Kh = qweight.shape
        K = Kh * 2
    elif qweight.dtype == torch.int32:
        N, Kw = qweight.shape
        K = Kw * 8
    else:
        raise TypeError("qweight must be int32 [N,K/8] or int8/uint8 [N,K/2]")
    if K % GROUP_SIZE:
        raise ValueError("K must be a multiple of 128")
    if group_size == K and K > 128:
        group_size = 0
    if group_size not in (0, 32, 64, 128):
        raise ValueError("group_size must be 32, 64, 128, or 0 / K (per-channel)")
    if signed and zeros is not None:
        raise ValueError("signed int4 is symmetric (W = q * s): zeros must be None")
    qweight = qweight.contiguous()
    G = K // group_size if group_size else 1
    sp = zp = None
    if scales is not None:
        if scales.shape != (N, G) or scales.dtype != torch.float16:
            raise ValueError(f"scales must be fp16 [{N},{G}]")
        scales = scales.contiguous(); sp = scales.data_ptr()
    if zeros is not None:
        if zeros.shape != (N, G) or zeros.dtype != torch.uint8:
            raise ValueError(f"zeros must be uint8 [{N},{G}]")
        zeros = zeros.contiguous(); zp = zeros.data_ptr()
    lib = L.load()
    nbytes = int(lib.sk_q4_bytes_ex(N, K, group_size))
    out = torch.empty(nbytes, dtype=torch.uint8, device=qweight.device)
    with torch.cuda.device(qweight.device):
        L.check(lib.sk_prepack_q4_ex(qweight.data_ptr(), sp, zp, N, K, group_size, 1 if signed else 0,
                                     out.data_ptr(), nbytes, _stream_ptr(qweight.device)), "sk_prepack_q4_ex")
    return PackedQ4(out, N, K, group_size, bool(signed))


def dequant_w4(QLB: PackedQ4) -> torch.Tensor:
    """W [N,K] fp16 = (q - z) * s, bit-exact with the fp16 expression evaluated on the CPU."""
    W = torch.empty((QLB.N, QLB.K), dtype=torch.float16, device=QLB.data.device)
    with torch.cuda.device(W.device):
        L.check(L.load().sk_dequant_q4_ex(QLB.data.data_ptr(), QLB.N, QLB.K, QLB.group_size, W.data_ptr(),
                                          W.stride(0), _stream_ptr(W.device)), "sk_dequant_q4_ex")
    return W


def streamk_fp16_ladder_block_reduce_q4(A, QLB: PackedQ4, *, fixup="block_reduce",
                                        schedule="auto", **kw):
    """W4A16: C = A @ ((q - z) * s).T, fp16 activations, uint4 weights.

    Mirrors `tl_mod(A, QLB, C)` of streamk_fp16_ladder_block_reduce_q4.py:143-599."""
    o = _options(kw)
    _check_matrix("A", A, torch.float16)
    if not isinstance(QLB, PackedQ4):
        raise TypeError("QLB must come from q4_prepack()")
    M, K = A.shape
    if K != QLB.K:
        raise ValueError(f"Incompatible dimensions: A {tuple(A.shape)} weight K={QLB.K}")
    A = _aligned16(_rowmajor(A))
    Cout = _out(o["out"], M, QLB.N, torch.float16, A.device)
    prob = _problem(M, QLB.N, K, A.stride(0), 0, Cout.stride(0), "nt", schedule, fixup, o)
    prob.flags |= L.SK_FLAG_Q4_GROUP[QLB.group_size]
    with _on(A.device):
        ws = _workspace(A.device)
        L.check(L.load().sk_gemm_w4a16(C.byref(prob), A.data_ptr(), QLB.data.data_ptr(),
                                       Cout.data_ptr(), ws.buf.data_ptr(), ws.nbytes,
                                       _stream_ptr(A.device)), "sk_gemm_w4a16")
    return Cout


# --------------------------------------------------------------------------- 8-bit integers
def int8_quantize(X: torch.Tensor, *, pdl: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of X [M,K] (fp16 or bf16) as 8-bit integers: (Q int8 [M,K], scale fp32 [M]).

    With a = max_k |X[m,k]|: scale[m] = a / 127 and Q[m,k] = 127 X[m,k] / a rounded to the
    nearest integer (halves to even, of the exact quotient), so X is about Q * scale[:, None].
    One scale per row: tokens when X holds activations, output channels when it holds a weight
    [N,K].  A row of zeros has scale 0; a row that holds a NaN or an infinity has scale NaN and
    Q = 0, so that products with it are NaN.  Q's row pitch is K rounded up to 16 bytes (what
    streamk_int8_nt reads without a copy).  Rows of X may be strided.  pdl: programmatic
    dependent launch (see _options(); here on unless switched off).  No autograd graph is recorded.
    No counterpart in the reference."""
    if pdl:
        r = (_fast or _load_fast()).quantize(X)
        if r is not None:
            return r
    _check_matrix("X", X, HALF_TYPES)
    M, K = X.shape
    if M < 1 or K < 1:
        raise ValueError(f"X must not be empty, got shape {(M, K)}")
    _check_int32(M=M, K=K, pitch=X.stride(0))
    X = _rowmajor(X)
    device = X.device
    pitch = -(-K // 16) * 16
    Q = torch.empty_strided((M, K), (pitch, 1), dtype=torch.int8, device=device)
    scale = torch.empty_strided((M,), (1,), dtype=torch.float32, device=device)
    flags = (L.SK_FLAG_BF16 if X.dtype == torch.bfloat16 else 0) | (L.SK_FLAG_PDL if pdl else 0)
    with _on(device):
        L.check(L.load().sk_quantize_i8(X.data_ptr(), M, K, X.stride(0) if M > 1 else K, flags, Q.data_ptr(), pitch,
                                        scale.data_ptr(), _stream_ptr(device)), "sk_quantize_i8")
    return Q, scale


def _check_int32(**extents) -> None:
    for name, v in extents.items():
        if v > 0x7fffffff:
            raise ValueError(f"{name} is {v}: extents and pitches are 32-bit numbers")


def _check_scale(name: str, s: torch.Tensor, n: int, device) -> torch.Tensor:
    if not isinstance(s, torch.Tensor) or s.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on the operands' device")
    if s.dtype != torch.float32:
        raise TypeError(f"{name} must be torch.float32, got {s.dtype}")
    if s.shape == (n,) and s.is_contiguous():
        return s
    if s.shape not in ((n,), (n, 1), (1, n)):
        raise ValueError(f"{name} must have {n} elements, got shape {tuple(s.shape)}")
    return s.reshape(n).contiguous()


def _rows16(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """An int8 matrix with 16-byte aligned rows (TMA), copied only if it has none, and its pitch."""
    ld, unit = t.stride()
    if unit == 1 and ld % 16 == 0 and ld >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t, ld
    n = torch.empty((t.shape[0], -(-t.shape[1] // 16) * 16), dtype=t.dtype, device=t.device)
    n[:, : t.shape[1]].copy_(t)
    return n, n.stride(0)


def streamk_int8_nt(A: torch.Tensor, B: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, *,
                    out_dtype: torch.dtype = torch.float16, schedule: str = "auto", **kw) -> torch.Tensor:
    """C = (A @ B.T) * scale_a[:, None] * scale_b[None, :] with 8-bit integer operands: A [M,K] and
    B [N,K] int8, scales fp32 [M] (tokens) and [N] (output channels), C fp16 or bf16.

    32-bit integer sums, exact whatever the schedule: every schedule returns the same bits.
    C = (float(sum) * scale_a) * scale_b, then one rounding to out_dtype.  K at most 131071.
    Operands whose rows are not 16-byte aligned are copied first.  Same schedules and keyword
    options as streamk_fp16_nt (see _options(); pdl is on unless switched off).  No autograd graph is
    recorded.  No counterpart in the reference."""
    if not kw and schedule == "auto" and out_dtype in HALF_TYPES:
        r = (_fast or _load_fast()).gemm_i8(A, B, scale_a, scale_b, out_dtype == torch.bfloat16)
        if r is not None:
            return r
    o = _options(kw)
    if o["pdl"] is None:
        o["pdl"] = True
    if out_dtype not in HALF_TYPES:
        raise TypeError(f"out_dtype must be one of {HALF_TYPES}, got {out_dtype}")
    o["_bf16"] = out_dtype == torch.bfloat16
    _check_matrix("A", A, torch.int8)
    _check_matrix("B", B, torch.int8)
    device = A.device
    if device != B.device:
        raise ValueError("A and B must be on the same device")
    M, K = A.shape
    N, Kb = B.shape
    if K != Kb:
        raise ValueError(f"Incompatible dimensions: A {tuple(A.shape)} B {tuple(B.shape)}")
    if M < 1 or N < 1 or K < 1:
        raise ValueError(f"operands must not be empty: A {tuple(A.shape)} B {tuple(B.shape)}")
    _check_int32(M=M, N=N, K=K, pitch_a=A.stride(0), pitch_b=B.stride(0))
    with _on(device):
        scale_a = _check_scale("scale_a", scale_a, M, device)
        scale_b = _check_scale("scale_b", scale_b, N, device)
        A, lda = _rows16(A)
        B, ldb = _rows16(B)
        Cout = _out(o["out"], M, N, out_dtype, device)
        prob = _problem(M, N, K, lda, ldb, Cout.stride(0), "nt", schedule, "block_reduce", o)
        ws, ws_bytes, ws_flags = _call_workspace(device)
        prob.flags |= ws_flags
        L.check(L.load().sk_gemm_i8(C.byref(prob), A.data_ptr(), B.data_ptr(), scale_a.data_ptr(), scale_b.data_ptr(),
                                    Cout.data_ptr(), ws, ws_bytes, _stream_ptr(device)), "sk_gemm_i8")
    return Cout


# --------------------------------------------------------------------------- grouped by expert
def _aligned16_batch(t: torch.Tensor) -> torch.Tensor:
    """[E, R, C] 16-bit weights with 16-byte aligned rows (TMA), copied only if they have none."""
    E, R, Cc = t.shape
    if (t.stride(2) == 1 and t.stride(1) >= Cc and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0
            and (E == 1 or (t.stride(0) >= R * t.stride(1) and t.stride(0) % 8 == 0))):
        return t
    n = torch.empty((E, R, -(-Cc // 8) * 8), dtype=t.dtype, device=t.device)
    n[:, :, :Cc].copy_(t)
    return n[:, :, :Cc]


def _grouped(kind, A, B, offsets, out, out_dtype, num_sms, timeout_us, pdl):
    if out is None and pdl and not (num_sms or timeout_us) and isinstance(A, torch.Tensor):
        fp32 = out_dtype is torch.float32
        if fp32 or out_dtype is None or out_dtype is A.dtype:
            r = (_fast or _load_fast()).grouped(L.GROUPED_KINDS[kind], A, B, offsets, fp32)
            if r is not None:
                return r
    _check_matrix("A", A, HALF_TYPES)
    dtype, device = A.dtype, A.device
    if not isinstance(B, torch.Tensor) or not B.is_cuda:
        raise ValueError("B must be a CUDA tensor (this library has no CPU path)")
    if B.dtype != dtype:
        raise TypeError(f"B must be {dtype} like A, got {B.dtype}")
    if not isinstance(offsets, torch.Tensor) or offsets.device != device or B.device != device:
        raise ValueError("A, B and offsets must be CUDA tensors on the same device")
    off64 = offsets.dtype == torch.int64
    if not off64 and offsets.dtype != torch.int32:
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    if offsets.dim() != 1 or offsets.shape[0] < 2:
        raise ValueError(f"offsets must be 1-D with one more element than there are groups, got shape {tuple(offsets.shape)}")
    T, K = A.shape
    E = offsets.shape[0] - 1
    bf16 = dtype == torch.bfloat16
    if kind == "tn":
        if B.dim() != 2 or B.shape[0] != T:
            raise ValueError(f"Incompatible dimensions: A {tuple(A.shape)} B {tuple(B.shape)}")
        N = B.shape[1]
        dtype = dtype if out_dtype is None else out_dtype
        if dtype not in (A.dtype, torch.float32):
            raise TypeError(f"out_dtype must be {A.dtype} or torch.float32, got {dtype}")
        shape = (E, K, N)
    else:
        if B.dim() != 3 or B.shape[0] != E or B.shape[2 if kind == "nt" else 1] != K:
            raise ValueError(f"Incompatible dimensions: A {tuple(A.shape)} B {tuple(B.shape)} and {E} groups")
        N = B.shape[1 if kind == "nt" else 2]
        shape = (T, N)
    if N < 1 or K < 1:
        raise ValueError(f"operands must not be empty: A {tuple(A.shape)} B {tuple(B.shape)}")
    _check_int32(T=T, N=N, K=K)
    if out is not None and (out.shape != shape or out.dtype != dtype or out.device != A.device or out.stride(-1) != 1
                            or out.stride(-2) < N or (kind == "tn" and E > 1 and out.stride(0) < K * out.stride(1))):
        raise ValueError(f"out must be a row-major {list(shape)} tensor of type {dtype} on A's device")
    with _on(device):
        if out is not None:
            Cout = out
        elif kind == "tn":
            Cout = torch.empty_strided(shape, (K * N, N, 1), dtype=dtype, device=device)
        else:
            Cout = torch.empty_strided(shape, (N, 1), dtype=dtype, device=device)
        if T == 0:
            return Cout.zero_() if kind == "tn" else Cout
        A = _aligned16(_rowmajor(A))
        B = _aligned16(_rowmajor(B)) if kind == "tn" else _aligned16_batch(B)
        if not offsets.is_contiguous():
            offsets = offsets.contiguous()
        flags = ((L.SK_FLAG_BF16 if bf16 else 0) | (L.SK_FLAG_PDL if pdl else 0)
                 | (L.SK_FLAG_OFFSETS_64 if off64 else 0) | (L.SK_FLAG_OUT_F32 if dtype == torch.float32 else 0)
                 | (L.SK_FLAG_ZERO_REST if out is None and kind != "tn" else 0))
        bs, cs = B.stride(), Cout.stride()
        prob = L.SkGroupedProblem(L.GROUPED_KINDS[kind], T, E, N, K, num_sms or 0, timeout_us or 0, flags,
                                  A.stride(0), bs[-2], cs[-2], 0 if kind == "tn" else bs[0], cs[0] if kind == "tn" else 0)
        ws, ws_bytes, ws_flags = _call_workspace(device)
        prob.flags |= ws_flags
        L.check(L.load().sk_gemm_grouped(C.byref(prob), A.data_ptr(), B.data_ptr(), offsets.data_ptr(), Cout.data_ptr(),
                                         ws, ws_bytes, _stream_ptr(device)), "sk_gemm_grouped")
    return Cout


def streamk_grouped_nt(A, B, offsets, *, out=None, num_sms=None, timeout_us=None, pdl=True):
    """C[t] = B[e] @ A[t] for the group e that row t belongs to: the linear layers of a set of
    experts.  A [T,K] and B [E,N,K] fp16 (or bf16), C [T,N] of the same type, fp32 accumulation.

    The rows of A are sorted by group: group e holds rows offsets[e] .. offsets[e+1]; offsets is
    an int32 or int64 CUDA tensor of E + 1 ascending numbers (nothing is read back by the host, so
    the call can be captured and replayed with other sizes).  Groups may be empty; there are at most
    1024.  Rows before offsets[0] and from offsets[E] on belong to no group: zero in a fresh result,
    left as they are in `out`, which shares no element with the operands.  Offsets out of order are
    clamped on the device and reported by check_status(), those of a replay as well.
    No autograd graph is recorded, here and in the two gradients, which are calls of their own:
    streamk_grouped_nn(dC, B, offsets) for A, streamk_grouped_tn(dC, A, offsets) for B.  Operands whose
    rows are not 16-byte aligned are copied first.  num_sms, timeout_us, pdl: see _options() (pdl is on unless switched off).  No counterpart in the reference."""
    return _grouped("nt", A, B, offsets, out, None, num_sms, timeout_us, pdl)


def streamk_grouped_nn(A, B, offsets, *, out=None, num_sms=None, timeout_us=None, pdl=True):
    """C[t] = A[t] @ B[e]: A [T,K], B [E,K,N], C [T,N].  The input gradient of streamk_grouped_nt
    (dA = streamk_grouped_nn(dC, B, offsets) with the same B [E,N,K]); otherwise the same rules."""
    return _grouped("nn", A, B, offsets, out, None, num_sms, timeout_us, pdl)


def streamk_grouped_tn(A, B, offsets, *, out=None, out_dtype=None, num_sms=None, timeout_us=None, pdl=True):
    """C[e] = sum over the rows t of group e of outer(A[t], B[t]): A [T,K], B [T,N], C [E,K,N], zero
    for an empty group.  The weight gradient of streamk_grouped_nt (dB = streamk_grouped_tn(dC, A,
    offsets)).  out_dtype: the operands' type (default) or torch.float32 (off by a few 2^-23 of the
    sums' norm, however many rows a group has).  Offsets as in streamk_grouped_nt; rows of no group,
    whatever they hold, do not count."""
    return _grouped("tn", A, B, offsets, out, out_dtype, num_sms, timeout_us, pdl)
