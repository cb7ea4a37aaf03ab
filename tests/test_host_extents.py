"""Extents and pitches beyond 32 bits are refused by the Python layer, not taken modulo 2^32 (the
fields of sk_problem are 32-bit numbers, and ctypes cuts what does not fit)."""
import pytest

import streamk_b200 as sk
from streamk_b200 import ops

OPTIONS = dict.fromkeys(ops._OPTION_KEYS)


@pytest.mark.parametrize("field", range(6))
@pytest.mark.parametrize("value", [1 << 31, (1 << 32) + 64, (1 << 40) + 64])
def test_problem(field, value):
    fields = [64] * 6                       # M, N, K, lda, ldb, ldc: a matrix in a very wide buffer, say
    ops._problem(*fields, "nt", "auto", "block_reduce", OPTIONS)
    fields[field] = value
    with pytest.raises(ValueError, match="32-bit"):
        ops._problem(*fields, "nt", "auto", "block_reduce", OPTIONS)


def test_the_largest_that_fits_is_kept():
    p = ops._problem(1, 2, 3, 0x7fffffff, 0x7ffffff0, 0x7fffffff, "nt", "auto", "block_reduce", OPTIONS)
    assert (p.M, p.N, p.K, p.lda, p.ldb, p.ldc) == (1, 2, 3, 0x7fffffff, 0x7ffffff0, 0x7fffffff)


@pytest.mark.parametrize("kind", ["f32", "f16", "w4a16", "int8"])
def test_schedule_info(kind):
    for shape in (((1 << 32) + 5, 256, 256), (5, (1 << 32) + 256, 256), (5, 256, (1 << 32) + 256)):
        with pytest.raises(ValueError, match="32-bit"):
            sk.schedule_info(*shape, kind=kind)
