"""A workspace of one size serves every smaller call: the sizes that are reported never fall
where rows, logits, tokens, sequences or the longest sequence grow, and are never below what
a call's plan lays out (CPU)."""
import ctypes as C
import random

import pytest

from inferno_hip import _lib
from test_gd_plan import LIB, of


@pytest.fixture(scope="module")
def lib():
    from inferno_hip import build
    build.build_checks()
    return C.CDLL(str(LIB))


def test_sampling(lib):
    lib.sample_plan_of.argtypes = [C.c_int] * 2 + [C.POINTER(C.c_longlong)]
    names = ("per", "slices", "rows", "bounds", "bins", "merged", "list", "bytes")
    size = _lib.lib().ihip_sample_scratch_bytes
    vocabs = sorted({1, 2, 700, 4096, 4097, 8192, 8193, 12288, 32000, 49152, 65536, 151936, 262144, (1 << 21) + 5, 1 << 22}
                    | {4096 * i + d for i in range(1, 30) for d in (0, 1)})
    last = dict.fromkeys(vocabs, 0)
    for rows in list(range(1, 130)) + [255, 256, 257, 511, 512, 513, 600, 5000]:
        before = 0
        for vocab in vocabs:
            n = size(rows, vocab)
            assert n >= max(before, last[vocab]), (rows, vocab)
            assert n >= of(lib.sample_plan_of, names, rows, vocab)["bytes"], (rows, vocab)
            before = last[vocab] = n
