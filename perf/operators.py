"""Cases of the 8-bit integer product, its quantiser, and the products grouped by expert.

Four operators, each in a plain form (elementary torch operations, 32 bits or more) and as a user
calls this library's kernels:

  quantize   q[m,k] = round(127 x[m,k] / a[m]), s[m] = a[m] / 127, a[m] = max_k |x[m,k]|
             (ties to even); rows of activations, one scale per token
  int8       C[m,n] = s_a[m] s_b[n] sum_k A[m,k] B[n,k], int8 operands
  grouped    Y[t,:] = W[e] X[t,:] for the expert e whose rows offsets[e] <= t < offsets[e+1] hold t;
             rows that belong to no expert are zero
  gradients  of the grouped product: dX[t,:] = W[e]^T dY[t,:], dW[e] = sum_t dY[t,:] X[t,:]^T

`own` chooses between the two; cases are dicts of plain values.
"""
import math

import numpy as np
import torch

own = False

if own:
    import streamk_b200  # noqa: F401

_DEVICE = "cuda"
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _quantize_case(name, M, K, dtype, pitch=0):
    return {"name": name, "op": "quantize", "M": M, "K": K, "dtype": dtype, "pitch": pitch}


def _int8_case(name, M, N, K, dtype):
    return {"name": name, "op": "int8", "M": M, "N": N, "K": K, "dtype": dtype}


def _grouped_case(name, op, T, rest, E, N, K, skew, dtype, grad="bf16"):
    return {"name": name, "op": op, "T": T, "rest": rest, "E": E, "N": N, "K": K, "skew": skew, "dtype": dtype,
            "grad": grad}


def listed():
    return [
        # the activations of a small decoding batch, ahead of an 8-bit layer
        _quantize_case("quantize_16x4096", 16, 4096, "fp16"),
        # a prompt batch of activations, rows of a wider buffer (two halves of a fused projection)
        _quantize_case("quantize_8192x11008", 8192, 11008, "bf16", 22016),
        # one decoded token through an 8-bit layer: a stream of the weights
        _int8_case("int8_1x11008x4096", 1, 11008, 4096, "fp16"),
        # a decoding batch, down projection
        _int8_case("int8_16x4096x11008", 16, 4096, 11008, "bf16"),
        # a chunk of a prompt with an odd number of tokens, fused projection
        _int8_case("int8_250x12288x4096", 250, 12288, 4096, "fp16"),
        # a full prompt batch through the largest layer of the benchmark
        _int8_case("int8_8192x28672x8192", 8192, 28672, 8192, "bf16"),
        # eight decoded tokens, two experts each, of eight: all the work is reading the experts used
        _grouped_case("grouped_16_e8_11008x4096", "grouped", 16, 0, 8, 11008, 4096, 0.5, "fp16"),
        # a decoding batch of 128 over 64 small experts, in a buffer of fixed size that it does not fill
        _grouped_case("grouped_250_e64_2048x4096", "grouped", 250, 6, 64, 2048, 4096, 0.7, "bf16"),
        # a prompt batch, two experts of eight per token, unevenly loaded
        _grouped_case("grouped_16384_e8_11008x4096", "grouped", 16384, 0, 8, 11008, 4096, 0.4, "bf16"),
        # gradients of a small layer on a short batch, some experts without a row
        _grouped_case("gradients_300_e16_1024x1024", "gradients", 300, 12, 16, 1024, 1024, 1.5, "fp16", "fp16"),
        # a training micro-batch over many experts, weight gradients accumulated elsewhere in fp32
        _grouped_case("gradients_4099_e32_2048x4096", "gradients", 4099, 0, 32, 2048, 4096, 0.6, "bf16", "fp32"),
        # a large training batch over eight experts
        _grouped_case("gradients_16384_e8_11008x4096", "gradients", 16384, 0, 8, 11008, 4096, 0.3, "bf16", "bf16"),
    ]


def _spread(rng, low, high, step=1):
    """A size between low and high, evenly over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quantize", "int8", "grouped", "gradients"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "quantize":
        M = _spread(rng, 1, 8192)
        K = _spread(rng, 256, 11008, 8)
        return {"op": op, "M": M, "K": K, "dtype": dtype, "pitch": rng.choice([0, K + 64, 2 * K])}
    if op == "int8":
        return {"op": op, "M": _spread(rng, 1, 8192), "N": _spread(rng, 256, 28672), "K": _spread(rng, 256, 8192, 16),
                "dtype": dtype}
    E = rng.choice([2, 5, 8, 16, 32, 64])
    T = _spread(rng, 1, 16384)
    N = _spread(rng, 256, 11008, 8)
    K = _spread(rng, 256, 4096, 8)
    while E * N * K > 8 * 11008 * 4096:   # no more weights than the largest listed case has
        E //= 2
    return {"op": op, "T": T, "rest": rng.choice([0, 0, 1, 37]), "E": E, "N": N, "K": K,
            "skew": rng.choice([0.0, 0.4, 0.8, 1.5]), "dtype": dtype, "grad": rng.choice([dtype, "fp32"])}


def _sizes(case):
    """Rows of each expert: shares falling as (i + 1) ** -skew, whole numbers that add up to T."""
    w = np.arange(1, case["E"] + 1, dtype=np.float64) ** -case["skew"]
    share = w / w.sum() * case["T"]
    n = np.floor(share).astype(np.int64)
    order = np.argsort(-(share - n), kind="stable")
    n[order[: case["T"] - int(n.sum())]] += 1
    return n


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape, scale=1.0):
        t = torch.empty(*shape, dtype=dtype, device=_DEVICE)
        t.normal_(0.0, scale, generator=g)
        return t

    if op == "quantize":
        M, K = case["M"], case["K"]
        # a few channels are far larger than the rest, as in the activations of a language model
        gain = torch.ones(K, dtype=torch.float32, device=_DEVICE)
        gain[torch.randint(0, K, (max(1, K // 512),), generator=g, device=_DEVICE)] = 20.0
        x = normal(M, max(K, case["pitch"]))[:, :K]
        x.mul_(gain.to(dtype))
        return {"op": op, "x": x}
    if op == "int8":
        M, N, K = case["M"], case["N"], case["K"]

        def quantized(rows, scale):
            # codes of a normal distribution whose largest value in the row sits at 127
            v = torch.empty(rows, K, dtype=torch.float16, device=_DEVICE)
            v.normal_(0.0, 1.0, generator=g)
            a = v.abs().amax(dim=1, keepdim=True)
            q = (v / a * 127).round_().to(torch.int8)
            s = (a.float().flatten() / 127) * scale
            return q, s

        A, sa = quantized(M, 1.0)
        B, sb = quantized(N, 0.02)
        return {"op": op, "A": A, "B": B, "sa": sa, "sb": sb, "dtype": dtype}
    E, N, K, T = case["E"], case["N"], case["K"], case["T"]
    sizes = _sizes(case)
    perm = torch.randperm(E, generator=torch.Generator().manual_seed(seed)).numpy()
    sizes = sizes[perm]
    bounds = np.concatenate([[0], np.cumsum(sizes)])
    state = {"op": op, "X": normal(T + case["rest"], K), "W": normal(E, N, K, scale=0.02),
             "offsets": torch.tensor(bounds, dtype=torch.int32, device=_DEVICE),
             "longest": int(sizes.max()), "dtype": dtype, "grad": _TYPES[case["grad"]]}
    if op == "gradients":
        state["dY"] = normal(T + case["rest"], N)
    return state


# ------------------------------------------------------------------------------ the plain forms
def _rows_of(offsets, longest):
    """[E, longest] row of each expert's i-th token, and whether it has one."""
    i = torch.arange(longest, device=offsets.device)
    rows = offsets[:-1, None].long() + i[None, :]
    return rows, rows < offsets[1:, None]


def _by_expert(t, offsets, longest):
    """[E, longest, width] fp32: the rows of each expert, padded with zeros."""
    rows, valid = _rows_of(offsets, longest)
    picked = t[rows.clamp(max=t.shape[0] - 1)].float()
    return torch.where(valid[:, :, None], picked, picked.new_zeros(()))


def _by_row(y, offsets, total):
    """The inverse of _by_expert: [total, width], zero where a row belongs to no expert."""
    r = torch.arange(total, device=offsets.device, dtype=offsets.dtype)
    e = torch.searchsorted(offsets[1:], r, right=True)
    some = (e < y.shape[0]) & (r >= offsets[0])
    e = e.clamp(max=y.shape[0] - 1)
    i = (r - offsets[e]).clamp(min=0, max=y.shape[1] - 1).long()
    picked = y[e, i]
    return torch.where(some[:, None], picked, picked.new_zeros(()))


def _plain_quantize(x):
    v = x.double()                        # (32 bits would move values that sit next to a half)
    a = v.abs().amax(dim=1)
    q = torch.round(v * 127 / a[:, None]).nan_to_num(0.0).to(torch.int8)
    return q, a.float() / 127


def _plain_int8(A, B, sa, sb, dtype):
    return ((A.float() @ B.float().T) * sa[:, None] * sb[None, :]).to(dtype)


def _plain_grouped(X, W, offsets, longest):
    y = _by_expert(X, offsets, longest) @ W.float().transpose(1, 2)
    return _by_row(y, offsets, X.shape[0]).to(X.dtype)


def _plain_gradients(dY, X, W, offsets, longest, grad):
    d = _by_expert(dY, offsets, longest)
    dX = _by_row(d @ W.float(), offsets, X.shape[0]).to(X.dtype)
    dW = (d.transpose(1, 2) @ _by_expert(X, offsets, longest)).to(grad)
    return dX, dW


def run(state):
    op = state["op"]
    if own:
        import streamk_b200 as sk
        if op == "quantize":
            return sk.int8_quantize(state["x"])
        if op == "int8":
            return sk.streamk_int8_nt(state["A"], state["B"], state["sa"], state["sb"], out_dtype=state["dtype"])
        if op == "grouped":
            return sk.streamk_grouped_nt(state["X"], state["W"], state["offsets"])
        return (sk.streamk_grouped_nn(state["dY"], state["W"], state["offsets"]),
                sk.streamk_grouped_tn(state["dY"], state["X"], state["offsets"], out_dtype=state["grad"]))
    if op == "quantize":
        return _plain_quantize(state["x"])
    if op == "int8":
        return _plain_int8(state["A"], state["B"], state["sa"], state["sb"], state["dtype"])
    if op == "grouped":
        return _plain_grouped(state["X"], state["W"], state["offsets"], state["longest"])
    return _plain_gradients(state["dY"], state["X"], state["W"], state["offsets"], state["longest"], state["grad"])


def work(case):
    op = case["op"]
    if op == "quantize":
        M, K = case["M"], case["K"]
        return {"bytes": 3 * M * K + 4 * M, "flops": 3 * M * K}
    if op == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K + N * K + 4 * (M + N) + 2 * M * N, "flops": 2 * M * N * K}
    E, N, K, T, R = case["E"], case["N"], case["K"], case["T"], case["rest"]
    used = int((_sizes(case) > 0).sum())
    if op == "grouped":
        return {"bytes": 2 * T * K + 2 * used * N * K + 2 * (T + R) * N + 4 * (E + 1), "flops": 2 * T * N * K}
    grad = 4 if case["grad"] == "fp32" else 2
    return {"bytes": 2 * T * (N + K) + 2 * used * N * K + 2 * (T + R) * K + grad * E * N * K + 4 * (E + 1),
            "flops": 4 * T * N * K}


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        # whole numbers are compared between the two forms; the scale has a value in 64 bits
        return None, torch.linalg.vector_norm(state["x"].double(), ord=math.inf, dim=1) / 127.0
    if op == "int8":
        total = torch.matmul(state["A"].to(torch.float64), state["B"].to(torch.float64).t())
        return total.mul_(state["sa"].double().unsqueeze(1)).mul_(state["sb"].double().unsqueeze(0))
    bounds = state["offsets"].tolist()
    X, W = state["X"], state["W"]
    if op == "grouped":
        Y = torch.zeros(X.shape[0], case["N"], dtype=torch.float64, device=X.device)
        for e in range(case["E"]):
            lo, hi = bounds[e], bounds[e + 1]
            if hi > lo:
                Y[lo:hi] = torch.einsum("tk,nk->tn", X[lo:hi].double(), W[e].double())
        return Y
    dY = state["dY"]
    dX = torch.zeros(X.shape[0], case["K"], dtype=torch.float64, device=X.device)
    dW = torch.zeros(case["E"], case["N"], case["K"], dtype=torch.float64, device=X.device)
    for e in range(case["E"]):
        lo, hi = bounds[e], bounds[e + 1]
        if hi > lo:
            dX[lo:hi] = torch.einsum("tn,nk->tk", dY[lo:hi].double(), W[e].double())
            dW[e] = torch.einsum("tn,tk->nk", dY[lo:hi].double(), X[lo:hi].double())
    return dX, dW
