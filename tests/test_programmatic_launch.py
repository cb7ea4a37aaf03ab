"""What programmatic dependent launch asks of the kernels, read from their sources.

A kernel launched that way is resident while the kernel before it in the stream still runs, and
waits for it with griddepcontrol.wait.  The faults that this makes possible show up on a GPU only by
chance, if at all, so the rules are checked in the text.
"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stream-k.tvm_b200", "csrc")


def _source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


def _kernels(text):
    """(signature, body and what follows) of every __global__ function."""
    for part in text.split("__global__")[1:]:
        signature, _, rest = part.partition("{")
        yield signature, rest


FILES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))
WAITING = [f for f in FILES if "griddep_wait()" in _source(f) and f.endswith(".cu")]


def test_the_waiting_kernels_are_found():
    assert {"sk_gemm_f16.cu", "sk_gemm_f16_2cta.cu", "sk_gemv.cu", "sk_grouped.cu", "sk_quant.cu",
            "sk_w4a16.cu"} <= set(WAITING)


@pytest.mark.parametrize("name", WAITING + [f for f in FILES if f.endswith(".cuh")])
def test_no_read_only_loads_of_what_a_predecessor_writes(name):
    """ld.global.nc is for data that nobody writes during the kernel's whole life; the operands of
    such a kernel may be the results of the one that is still running."""
    text = _source(name)
    assert "global.nc" not in text and "__ldg" not in text
    for signature, body in _kernels(text):
        if "griddep_wait()" in body:
            assert not re.search(r"const\s+[\w:]+\s*\*\s*__restrict__", signature), signature.strip()[:80]
