"""How the paged attention is launched (kv_attn_plan.h, through
tests/native/attn_plan_check.hip, on the CPU): the batches of the GPU tests reach
the variants that they are meant for, and the workspace and the counts hold what
a launch uses."""
import ctypes as C
import random
from pathlib import Path

import pytest

import kv_variants
from inferno_hip import _lib
from test_kv_refusals import batch, cache

LIB = Path(__file__).resolve().parent / "native" / "_build" / "libsdig_check.so"
TYPES = [(_lib.F32, _lib.F16), (_lib.F32, _lib.BF16), (_lib.F16, _lib.F16), (_lib.BF16, _lib.BF16)]


@pytest.fixture(scope="module")
def plan():
    from inferno_hip import build
    build.build_checks()
    fn = C.CDLL(str(LIB)).attn_plan_of
    fn.argtypes = [C.c_int] * 7 + [C.c_longlong, C.c_int, C.POINTER(C.c_longlong)]

    def of(act, kv, heads, kv_heads, dim, sequences, tokens, capacity, window=0):
        out = (C.c_longlong * 6)()
        fn(act, kv, heads, kv_heads, dim, sequences, tokens, capacity, 0 if window >= capacity else window, out)
        return dict(zip(("rows", "tiles", "parts", "least", "halves", "bytes"), out))
    return of


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("v", kv_variants.ALL, ids=kv_variants.Variant.ids)
def test_the_batches_reach_their_variants(plan, act, kv, v):
    for dim in v.dims:
        p = plan(act, kv, v.heads, v.kv_heads, dim, len(v.new), sum(v.new), 16 * v.width, v.window)
        assert p["rows"] == v.rows and v.parts[0] <= p["parts"] <= v.parts[1], p
        if v.rows == 128:
            assert bool(p["halves"]) == v.halves, p


def test_workspace_and_counts_hold_every_launch(plan):
    """Tiles of any batch of these sizes fit the plan's; counts are used for fewer tiles than there are; the
    workspace asked for holds every q type and window."""
    rng = random.Random(1)
    for _ in range(3000):
        kv_heads, group = rng.choice([1, 2, 8, 40, 300]), rng.choice([1, 3, 4, 16])
        sequences, tokens = rng.randint(1, 80), int(2 ** rng.uniform(0, 14))
        dim, width = 8 * rng.randint(1, 32), int(2 ** rng.uniform(0, 14))
        act, kv = rng.choice(TYPES)
        window = rng.choice([0, rng.randint(1, 16 * width)])
        p = plan(act, kv, kv_heads * group, kv_heads, dim, sequences, tokens, 16 * width, window)
        cuts = sorted(rng.randint(0, tokens) for _ in range(sequences - 1))
        new = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
        assert sum(-(-n * group // p["rows"]) for n in new) <= p["tiles"]
        assert p["parts"] == 1 or p["rows"] == 128 or p["tiles"] * kv_heads <= 4096
        floats = p["parts"] * tokens * kv_heads * group * (dim + 2)
        assert p["bytes"] == (0 if p["parts"] == 1 else 16384 + 4 * floats)
        c = cache(pages=1 << 20, type=kv, kv_heads=kv_heads, head_dim=dim, page_stride=kv_heads * 16 * dim)
        b = batch(sequences=sequences, tokens=tokens, table_stride=width)
        assert _lib.lib().ihip_attn_paged_scratch_bytes(act, kv_heads * group, C.byref(c), C.byref(b)) >= p["bytes"]
