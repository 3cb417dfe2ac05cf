"""How calls of the gated delta rule and of sampling are laid out (gd_plan.h and
sample_plan.h, through tests/native/gd_plan_check.hip, on the CPU): every chunk of any
batch has a number of its own within the plan's, areas do not overlap, and slices
cover a row."""
import ctypes as C
import random
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parent / "native" / "_build" / "libsdig_check.so"


@pytest.fixture(scope="module")
def lib():
    from inferno_hip import build
    build.build_checks()
    return C.CDLL(str(LIB))


def of(fn, names, *args):
    out = (C.c_longlong * 8)()
    fn(*[C.c_longlong(a) if a > 1 << 30 else a for a in args], out)
    return dict(zip(names, out))


def delta(lib, *args):
    lib.delta_plan_of.argtypes = [C.c_int] * 5 + [C.c_longlong] * 2 + [C.c_int, C.POINTER(C.c_longlong)]
    return of(lib.delta_plan_of, ("chunks", "steps", "tiles", "frag", "tri", "rows", "raw", "bytes"), *args)


def numbers(starts):
    """Of the chunks of 64 rows of every sequence, as the kernels form them."""
    return [(a >> 6) + s + c for s, (a, b) in enumerate(zip(starts, starts[1:])) for c in range(-(-(b - a) // 64))]


def test_chunks_have_numbers_of_their_own(lib):
    rng = random.Random(1)
    for _ in range(4000):
        sequences, tokens = rng.randint(1, 90), int(2 ** rng.uniform(0, 13))
        starts = sorted(rng.randint(0, tokens) for _ in range(sequences + 1))
        got = numbers(starts)
        p = delta(lib, 1, 2, 4, 64, 64, tokens, sequences, 0)
        assert len(set(got)) == len(got)
        if p["chunks"]:
            assert max(got, default=0) < p["tiles"]
        # a number's sequence is the last one that does not start behind it
        base = [(a >> 6) + s for s, a in enumerate(starts[:-1])]
        for t in got:
            s = max(i for i, b in enumerate(base) if b <= t)
            assert (t - base[s]) * 64 < starts[s + 1] - starts[s]


def test_areas_of_the_delta_rule(lib):
    rng = random.Random(2)
    for _ in range(1000):
        parts, k_heads, group = rng.choice([1, 2]), rng.randint(1, 20), rng.randint(1, 5)
        dk, dv = 16 * rng.randint(1, 8), 16 * rng.randint(1, 8)
        tokens, sequences = int(2 ** rng.uniform(0, 14)), rng.randint(1, 80)
        few = min(max(sequences * k_heads * group // 4, 10), 32)
        most = rng.choice([0, 1, 10, 11, few, few + 1, tokens])
        p = delta(lib, parts, k_heads, k_heads * group, dk, dv, tokens, sequences, most)
        longest = min(most or tokens, tokens)
        assert bool(p["chunks"]) == (longest > few) and bool(p["steps"]) == (longest <= few or sequences > 1)
        if not p["chunks"]:
            assert p["bytes"] == 0
            continue
        kd = 64 if dk <= 64 else 128
        assert p["frag"] == 64 * kd * 2 * parts
        assert p["tri"] == p["tiles"] * k_heads * 2 * p["frag"]
        assert p["rows"] - p["tri"] == p["tiles"] * k_heads * group * (6 * 2 * 1024 + kd * 64 * 2 * 2)
        assert p["raw"] - p["rows"] >= p["tiles"] * k_heads * group * 129 * 4
        assert p["bytes"] - p["raw"] == (4 * tokens * k_heads * group * dv if parts == 1 else 0)
        assert all(p[k] % 16 == 0 for k in ("tri", "rows", "raw"))


def test_slices_and_areas_of_sampling(lib):
    lib.sample_plan_of.argtypes = [C.c_int] * 2 + [C.POINTER(C.c_longlong)]
    rng = random.Random(3)
    for _ in range(3000):
        rows, vocab = int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 22))
        p = of(lib.sample_plan_of, ("per", "slices", "rows", "bounds", "bins", "merged", "list", "bytes"), rows, vocab)
        assert p["per"] in (4096, 8192) and (p["slices"] - 1) * p["per"] < vocab <= p["slices"] * p["per"]
        assert p["slices"] <= 512 and p["rows"] == min(rows, 256)
        n = p["rows"]
        assert p["bounds"] >= n * p["slices"] * 24 and p["bins"] - p["bounds"] == n * 64
        assert p["merged"] - p["bins"] == n * p["slices"] * 1024 * 12 and p["list"] - p["merged"] == n * 1024 * 12
        assert p["bytes"] - p["list"] == n * 4096 * 8
        assert all(p[k] % 16 == 0 for k in ("bounds", "bins", "merged", "list"))
