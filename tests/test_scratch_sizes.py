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


def test_the_delta_rule(lib):
    lib.delta_plan_of.argtypes = [C.c_int] * 5 + [C.c_longlong] * 2 + [C.c_int, C.POINTER(C.c_longlong)]
    rng = random.Random(5)

    def size(type_, K, H, dk, dv, tokens, sequences, most):
        layer = _lib.DeltaLayerStruct(state=1 << 30, slot_stride=H * dk * dv, slots=1, k_heads=K, v_heads=H, k_dim=dk, v_dim=dv,
                                      decay=1 << 20, dt_bias=1 << 21, norm_w=None, norm_eps=0.0, l2_eps=0.0, scale=1.0)
        batch = _lib.StateBatchStruct(q_starts=1, kv_lens=None, slots=1, sequences=sequences, tokens=tokens, most=most)
        return _lib.lib().ihip_gated_delta_scratch_bytes(type_, C.byref(layer), C.byref(batch))

    names = ("chunks", "steps", "tiles", "frag", "tri", "rows", "raw", "bytes")
    for _ in range(4000):
        K = rng.choice([1, 2, 8, 16])
        shape = K, K * rng.randint(1, 4), 16 * rng.randint(1, 8), 16 * rng.randint(1, 8)
        tokens, sequences = int(2 ** rng.uniform(0, 9)), int(2 ** rng.uniform(0, 7))
        most = rng.choice([0, rng.randint(1, 80)])
        less = (rng.randint(1, tokens), rng.randint(1, sequences), rng.randint(1, most) if most else rng.choice([0, rng.randint(1, 600)]))
        type_ = rng.choice([_lib.F32, _lib.F16, _lib.BF16])
        n = size(type_, *shape, tokens, sequences, most)
        assert n >= size(type_, *shape, *less), (shape, tokens, sequences, most, less)
        p = of(lib.delta_plan_of, names, 2 if type_ == _lib.F32 else 1, *shape, tokens, sequences, most)
        assert n >= p["bytes"]
    assert size(_lib.BF16, 16, 32, 128, 128, 61, 61, 1) == 0  # single tokens need none
