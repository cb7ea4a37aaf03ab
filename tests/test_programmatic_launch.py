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


@pytest.mark.parametrize("name", [f for f in WAITING if "tmem_alloc" in _source(f)])
def test_the_next_kernel_is_let_in_after_the_tensor_memory_is_allocated(name):
    """Let in before, the next kernel's CTAs could take the columns and wait for this kernel, whose
    allocation would wait for them."""
    found = 0
    for _, body in _kernels(_source(name)):
        alloc = [m.end() for m in re.finditer(r"\btmem_alloc(_pair)?\(", body)]
        let_in = [m.start() for m in re.finditer(r"griddep_launch_dependents\(", body)]
        if not alloc:
            continue
        found += 1
        assert len(alloc) == 1 and len(let_in) == 1 and let_in[0] > alloc[0]
        # in the allocating warp's own block, behind the instruction, so in its program order
        assert "}" not in body[alloc[0]:let_in[0]]
    assert found > 0
